// Penalties, biases and masks on a batch's logits, and the highest one left
// (include/zg_hip.h, zg_logits_adjust_device).
//
// A row's logits are read and written once.  Only the tokens in the history
// and the biases change, so a workgroup gathers those of its slice of the
// vocabulary in LDS and lists them, a thread forms the new value of each, in
// 64 bits and rounded once, and the values are laid over the logits on their
// way from registers to memory.  A history is read by every slice's
// workgroup, which keeps a few tokens of each hundred: a wave first packs
// those together (a ballot and a count of lower lanes, no atomics) and then
// takes them a lane each.  The count of a token is a sum of integers and the
// list's order of no account, so the order of the LDS atomics does not matter;
// the biases of one token are summed in their order.
//
// The bytes of 32 rows of 151936 take 6.4 us at 6.1 TB/s, a copy through this
// kernel with a mask 11.4; 500 tokens of history make it 14.2 us and 2500 15.6:
// barriers and shared memory between a slice's loads and its stores.  With 64
// rows of 9000 tokens 29 us: the histories, 38 slices of each row reading them
// from the L2s, are then 88 MB beside the logits' 39, and each of the eight L2s
// fetches them (38 MB fetched in all where 22 are there).
#include "zg_paged.hpp"

namespace zg {

// A token's word: it is in the history; it has a bias; it has several; the
// other bits count its generated occurrences (a history holds at most 2^28).
constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u, kSeveral = 0x20000000u, kCount = kSeveral - 1;
constexpr int kLeastSlice = 1024;
constexpr int kBatch = 8;    // history loads of a thread under way
constexpr int kList = 1024;  // listed tokens of a slice; where there are more, all are looked at

// A candidate of the greedy readout: the higher value wins, of equal ones the
// lower index.  Index -1: none.
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

template <bool BF16>
__device__ __forceinline__ float load_logit(const void* p, size_t at) {
    if constexpr (BF16) return bf16_to_f32(((const uint16_t*)p)[at]);
    else return ((const float*)p)[at];
}

// `more` and the lanes before this one that are in `lanes`.
__device__ __forceinline__ int lanes_before(uint64_t lanes, int more) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, (uint32_t)more));
}

// Workgroup (slice, row) of T threads and 4 V tokens a thread, four
// neighbouring ones at a time.  WHOLE: four logits are loaded and stored at
// once, which the rows' alignment must allow.
template <bool BF16, bool WHOLE, int T, int V>
__global__ __launch_bounds__(T) void logits_adjust_kernel(LogitArgs a, int slices) {
    constexpr int SLICE = 4 * T * V, WAVES = T / 64;
    static_assert(SLICE <= 32768, "offsets and a flag in 16 bits");
    __shared__ __align__(16) uint32_t value[SLICE];   // a token's word, then its new value
    __shared__ uint32_t touched[SLICE / 32];          // the listed tokens
    __shared__ uint16_t list[kList];
    __shared__ uint16_t hits[WAVES][64 * kBatch];     // a wave's history tokens in the slice, top bit: generated
    __shared__ uint16_t bias_of[SLICE];               // one of a token's biases
    __shared__ int listed;
    __shared__ Best found[WAVES];
    const size_t r = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const zg_logit_rules& u = a.rules;
    const size_t first = (size_t)blockIdx.x * SLICE;
    const int n = (int)min((size_t)SLICE, a.vocab - first);
    const size_t in = r * a.ld + first, out = r * a.out_ld + first;

    // Everything that does not hang on something else is asked for at once: the
    // row's numbers, the first of its history and biases (as much of them as
    // their strides hold, whatever their lengths say) and the logits.
    const int held = u.history ? u.history_lengths[r] : 0;
    const int prompt = u.prompt_lengths ? u.prompt_lengths[r] : 0;
    const int given = u.bias_ids ? u.bias_lengths[r] : 0;
    const float rep = u.repetition ? u.repetition[r] : 1.0f;
    const float freq = u.frequency ? u.frequency[r] : 0.0f, pres = u.presence ? u.presence[r] : 0.0f;
    const int mask_row = u.masks ? u.mask_of ? u.mask_of[r] : (int)r : -1;
    const int32_t* const history = u.history + (u.history ? r * u.history_stride : 0);
    const int room = u.history ? (int)u.history_stride : 0;
    uint32_t id[kBatch];
    auto load_history = [&](int from) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int i = from + k * T + tid;
            id[k] = i < room ? (uint32_t)history[i] : 0xffffffffu;
        }
    };
    load_history(0);
    const int32_t* const ids = u.bias_ids + (u.bias_ids ? r * u.bias_stride : 0);
    const float* const add = u.bias_values + (u.bias_ids ? r * u.bias_stride : 0);
    const uint32_t bias_id = u.bias_ids && tid < (int)u.bias_stride ? (uint32_t)ids[tid] : 0xffffffffu;
    v4f x[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int i = 4 * (k * T + tid);
        x[k] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (i < n) {
            if (WHOLE && i + 4 <= n) x[k] = load4<BF16>(a.logits, in + i);
            else
                for (int j = 0; j < 4; ++j)
                    if (i + j < n) x[k][j] = load_logit<BF16>(a.logits, in + i + j);
        }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) *(v4u*)&value[4 * (k * T + tid)] = v4u{0, 0, 0, 0};
    if (tid < SLICE / 32) touched[tid] = 0;
    if (tid == 0) listed = 0;
    const bool none = mask_row >= 0 && (size_t)mask_row >= u.mask_rows;  // a mask that is not there allows nothing
    const uint32_t* mask = mask_row >= 0 && !none ? u.masks + (size_t)mask_row * u.mask_stride + first / 32 : nullptr;
    uint32_t allowed[V];  // of the four tokens, and of those past the vocabulary none
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int i = 4 * (k * T + tid);
        allowed[k] = none || i >= n ? 0u : mask ? mask[i >> 5] >> (i & 31) : 0xfu;
        if (i + 4 > n && i < n) allowed[k] &= (1u << (n - i)) - 1;
    }
    if (held < 0) return;
    const int biases = u.bias_ids ? max(0, min(given, (int)u.bias_stride)) : 0, tokens = min(held, room);
    const bool changes = tokens > 0 || biases > 0;
    const int made_from = max(0, min(prompt, tokens)) - 64 * wave;  // less the wave's part of a token's place
    if (changes) {
        __syncthreads();
        auto enlist = [&](uint32_t at) {
            const uint32_t bit = 1u << (at & 31);
            if (atomicOr(&touched[at >> 5], bit) & bit) return;
            const int k = atomicAdd(&listed, 1);
            if (k < kList) list[k] = (uint16_t)at;
        };
        for (int from = 0; from < tokens; from += kBatch * T) {
            if (from + kBatch * T > tokens)  // the last ones: what is past the end is no token
#pragma unroll
                for (int k = 0; k < kBatch; ++k)
                    if (from + k * T + tid >= tokens) id[k] = 0xffffffffu;
            int got = 0;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const uint32_t at = id[k] - (uint32_t)first;  // below n: it is in the vocabulary
                const bool hit = at < (uint32_t)n;
                const uint64_t lanes = __ballot(hit);
                if (hit) hits[wave][lanes_before(lanes, got)] = (uint16_t)(at | (lane >= made_from - from - k * T ? 0x8000u : 0u));
                got += __popcll(lanes);
            }
            if (from + kBatch * T < tokens) load_history(from + kBatch * T);
            same_wave();
            for (int k = lane; k < got; k += 64) {
                const uint32_t at = hits[wave][k] & 0x7fffu, made = hits[wave][k] >> 15;
                enlist(at);
                // the top bit is set by or, not by sum: it is there once
                atomicOr(&value[at], kSeen);
                if (made) atomicAdd(&value[at], 1u);
            }
            same_wave();
        }
        // any of a token's biases stays in bias_of; the others then find it
        // there and mark the token
        auto each_bias = [&](auto then) {
            for (int i = tid; i < biases; i += T) {
                const uint32_t at = (i < T ? bias_id : (uint32_t)ids[i]) - (uint32_t)first;
                if (at < (uint32_t)n) then(i, at);
            }
        };
        each_bias([&](int i, uint32_t at) {
            enlist(at);
            atomicOr(&value[at], kBiased);
            bias_of[at] = (uint16_t)i;
        });
        __syncthreads();
        if (biases) {
            each_bias([&](int i, uint32_t at) {
                if (bias_of[at] != i) atomicOr(&value[at], kSeveral);
            });
            __syncthreads();
        }
#pragma unroll 1
        for (int k = tid; k < (listed <= kList ? listed : n); k += T) {
            const int i = listed <= kList ? list[k] : k;
            if (!(touched[i >> 5] >> (i & 31) & 1u)) continue;
            const uint32_t c = value[i];
            double v = (double)load_logit<BF16>(a.logits, in + i);
            if (c & kSeen) v = v > 0.0 ? v / (double)rep : v * (double)rep;
            if (c & kCount) v = v - (double)freq * (double)(c & kCount) - (double)pres;
            if (c & kSeveral) {
                double sum = 0.0;
                for (int j = 0; j < biases; ++j)
                    if (ids[j] == (int)(first + i)) sum += (double)add[j];
                v += sum;
            } else if (c & kBiased) {
                v += (double)add[bias_of[i]];
            }
            value[i] = BF16 ? (uint32_t)to_bf16(v) << 16 : __float_as_uint((float)v);
        }
        __syncthreads();
    }

    Best best{-INFINITY, -1};  // indices ascend: a later one takes a higher value
    bool odd = false;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int i = 4 * (k * T + tid);
        if (changes) {
            const uint32_t t = touched[i >> 5] >> (i & 31);
            const v4u w = *(const v4u*)&value[i];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (t >> j & 1u) x[k][j] = __uint_as_float(w[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!(allowed[k] >> j & 1u)) x[k][j] = -INFINITY;
            odd |= !(x[k][j] < INFINITY);
            if (x[k][j] > best.v) best = Best{x[k][j], (int)first + i + j};
        }
        if (i >= n) continue;
        if (WHOLE && i + 4 <= n) {
            if constexpr (BF16)  // the values are bfloat16 already
                *(uint2*)((uint16_t*)a.out + out + i) =
                    make_uint2(__builtin_amdgcn_perm(__float_as_uint(x[k][1]), __float_as_uint(x[k][0]), 0x07060302u),
                               __builtin_amdgcn_perm(__float_as_uint(x[k][3]), __float_as_uint(x[k][2]), 0x07060302u));
            else
                store4<false>(a.out, out + i, x[k]);
        } else {
            for (int j = 0; j < 4; ++j) {
                if (i + j >= n) break;
                if constexpr (BF16) ((uint16_t*)a.out)[out + i + j] = (uint16_t)(__float_as_uint(x[k][j]) >> 16);
                else ((float*)a.out)[out + i + j] = x[k][j];
            }
        }
    }
    if (a.status && __any(odd) && lane == 0) atomicOr(a.status, ZG_STATUS_NONFINITE);
    if (!a.greedy) return;
    best = wave_best(best);
    if (lane == 0) found[wave] = best;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < WAVES; ++w) best = better(best, found[w]);
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

static int slices_of(size_t vocab, int slice) { return (int)((vocab + slice - 1) / slice); }

size_t logits_workspace(size_t rows, size_t vocab) { return rows * slices_of(vocab, kLeastSlice) * sizeof(Best); }

template <bool BF16, bool WHOLE>
static int adjust(const LogitArgs& a, hipStream_t st) {
    // Every slice reads the row's history, so few long slices cost less, while
    // one row alone wants many short ones: with a vocabulary of 151936 slices
    // of 1024 and of 4096 tokens take 5.9 and 6.8 us at 1 row (600 tokens of
    // history), 8.6 and 7.2 at 3 (4000), 9.0 and 8.0 at 8 (2000), 21.5 and 17.0
    // at 32 (2500); slices of 8192, two workgroups to a CU, 19.6 at 32.
    const int slice = a.rows * slices_of(a.vocab, 4096) >= 96 ? 4096 : kLeastSlice, slices = slices_of(a.vocab, slice);
    const dim3 grid(slices, (unsigned)a.rows);
    // Of 512 threads 1024 workgroups run at once, of 256 the LDS holds 1280: the
    // latter are taken where they need fewer rounds, which pays if it halves
    // them, and of 16-bit logits wherever it spares one; but each thread then
    // has twice the history, so the longer that may be, the less.  us with 512
    // and 256 threads, a vocabulary of 151936, 600, 2500, 9000, 16000 tokens of
    // history: 27 rows (1026 slices) 16.1 15.1, 16.4 16.1, 19.2 19.6, 21.6 23.3;
    // 32 rows (1216) 18.3 16.4, 18.6 17.6, 21.3 20.9, 24.4 24.7, 16-bit 17.6 14.8,
    // 17.9 15.5, 20.7 19.4, 23.8 23.3; 64 rows (2432: 3 and 2 rounds) 26.3 25.4,
    // 26.5 26.7, 30.3 32.9, 16-bit 25.1 23.0, 25.4 24.2, 29.9 30.8; 101 rows (3838:
    // 4 and 3) 39.8 41.7, 39.4 42.6, 16-bit 33.8 31.7, 34.4 33.2, 41.1 42.2.  In as
    // many rounds: 34 rows (1292) 18.9 20.5, 16-bit 18.1 18.8; 26 (988) 14.4 15.1.
    constexpr size_t kMoreHistory = 18432;
    const size_t all = a.rows * slices, rounds = (all + 1023) / 1024, fewer = (all + 1279) / 1280;
    const size_t history = a.rules.history ? a.rules.history_stride : 0;
    if (slice == 4096 && fewer < rounds && (BF16 || fewer == 1) && history * rounds <= kMoreHistory)
        logits_adjust_kernel<BF16, WHOLE, 256, 4><<<grid, 256, 0, st>>>(a, slices);
    else if (slice == 4096) logits_adjust_kernel<BF16, WHOLE, 512, 2><<<grid, 512, 0, st>>>(a, slices);
    else logits_adjust_kernel<BF16, WHOLE, 256, 1><<<grid, 256, 0, st>>>(a, slices);
    return slices;
}

hipError_t logits_adjust(const LogitArgs& a, hipStream_t st) {
    // four logits at once where every row starts at a multiple of four
    const size_t four = a.bf16 ? 8 : 16;
    const bool whole = ((uintptr_t)a.logits | (uintptr_t)a.out) % four == 0 && a.ld % 4 == 0 && a.out_ld % 4 == 0;
    const int slices = a.bf16 ? (whole ? adjust<true, true>(a, st) : adjust<true, false>(a, st))
                              : (whole ? adjust<false, true>(a, st) : adjust<false, false>(a, st));
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.greedy) return e;
    logits_greedy_kernel<<<(unsigned)a.rows, 64, 0, st>>>(a, slices);
    return hipGetLastError();
}

}  // namespace zg

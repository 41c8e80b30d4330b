// Attention of a batch over a shared prefix and each row's own pages
// (include/zg_hip.h, zg_paged_attn_device).
//
// With s_t = scale q.k_t, out = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m) for
// any m, so a set of tokens is summed up by (m, l = sum e^(s_t - m), o = sum
// e^(s_t - m) v_t), and two sets join by scaling the one to the other's m.
// Work is cut into tiles of 32 tokens (16 of a 32-bit cache, the same bytes);
// a launch leaves such a triple per (row, kv head) and piece, and a second
// launch joins them.
//
// A wave takes a tile and 16 queries (columns: the query heads of one kv
// head; over the prefix also those of other rows) through the matrix cores
// without leaving its registers:
//   S^T [token][query] = K Q^T  -- the key rows are the first operand as they
//     lie in memory, 16 bytes a lane;
//   a lane then holds 8 scores (4) of one query, of tokens 16 (j / 4) + 4
//     quarter + j % 4, the order in which the second product takes them:
//   O^T [element][query] += V^T P^T -- value rows are loaded 16 bytes a lane
//     and transposed between a lane's own registers, 8 rows at a time (32-bit
//     rows need not be).
// So the tile needs neither LDS nor a barrier.
#include <algorithm>
#include <cmath>

#include "zg_paged.hpp"

namespace zg {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

constexpr int kCus = 256;
// Waves over the rows' own tiles: one per SIMD, since a tile's loads are all under
// way at once (8 rows of 32768 tokens 101 us = 5.3 TB/s) and every wave leaves
// pieces to join.  With 2048 one row of 32768 took 18.1 + 8.9 us for 17.4 + 6.2,
// 24 rows of up to 16384 24.4 + 7.2 for 22.3 + 5.7, 32 of up to 4096 with
// 64-element heads 47.4 for 43.6, only 200 short rows of those 35.7 for 40.5.
constexpr int kOwnWaves = 1024;
static_assert(kOwnWaves <= 4 * kCus, "paged_attn_workspace counts a workgroup to a CU");
constexpr size_t kOwnLds = 128 << 10; // for the staged queries of a workgroup's waves
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kRaise = 8.0f;      // log2: how far a score may pass the reference before sums are rescaled

template <bool IO, bool KV, int D>
struct Form {
    // a 32-bit query enters a bfloat16 product as three parts of 8 bits, its
    // 24 in all; so do the weights of 32-bit outputs.  16-bit outputs take two
    // parts of a weight: at most 2^-16 of it is left out, so at most 2^-16 of
    // sum w |v|, which is a 256th of the output's own rounding where the terms
    // do not cancel and as much as that where they leave a 256th of themselves
    // (24 rows of up to 16384 random tokens: 0.4% of the outputs a step from
    // the nearest, with 32-bit weights 0.05%).
    static constexpr int kParts = KV ? (IO ? 1 : 3) : 1;
    // the scale (in log2) is put on the queries, but for those that enter as
    // the bfloat16 they are
    static constexpr bool kScaled = !(KV && IO);
    static constexpr int kWeightParts = KV ? (IO ? 2 : 3) : 1;
    static constexpr int kSteps = KV ? D / 32 : D / 16;                // 16 bytes of a key per lane and step
    static constexpr int kWide = KV ? (D / 16 < 8 ? D / 16 : 8) : 4;   // elements of a value row per lane and load
    static constexpr int kLoads = D / (16 * kWide);
    static constexpr int kFrags = D / 16;                              // accumulators per 16 queries
    static constexpr int kHalves = KV ? 2 : 1;                         // 16 tokens each
    static constexpr int kTile = 16 * kHalves;
    static constexpr int kMine = 4 * kHalves;                          // of a tile's tokens, scores per lane and query
};

// The first 16 bits of two floats as a register of two bfloat16.
__device__ __forceinline__ uint32_t pack_high(float lo, float hi) {
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ float high_part(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

__device__ __forceinline__ v4f mfma_bf16(v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

// Queries in LDS in operand order, 16 bytes per (step, part, quarter, query):
// a wave's read is contiguous.  `who` gives query m's elements in memory.
template <bool IO, bool KV, int D, typename Who>
__device__ __forceinline__ void stage_queries(v4u* lds, int n, int thread, int threads, float to_log2, Who who) {
    using F = Form<IO, KV, D>;
    constexpr int E = KV ? 8 : 4;
    for (int i = thread; i < n * (D / E); i += threads) {
        const int m = i % n, c = i / n;
        const size_t at = who(m) + c * E;
        if constexpr (!KV) {
            lds[c * n + m] = __builtin_bit_cast(v4u, load4<IO>(who.base, at) * to_log2);
        } else if constexpr (IO) {
            lds[c * n + m] = *(const v4u*)((const uint16_t*)who.base + at);
        } else {
            v4f x[2] = {load4<false>(who.base, at) * to_log2, load4<false>(who.base, at + 4) * to_log2};
#pragma unroll
            for (int p = 0; p < F::kParts; ++p) {
                v4u w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = pack_high(x[j >> 1][(2 * j) & 3], x[j >> 1][(2 * j + 1) & 3]);
                lds[((c / 4 * F::kParts + p) * 4 + (c & 3)) * n + m] = w;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j >> 2][j & 3] -= high_part(x[j >> 2][j & 3]);
            }
        }
    }
}

// A wave's running sums for 16 queries: lane l holds query l % 16; o[f][r] is
// element 16 W g + W (4 quarter + r) + i of it, f = W g + i.
template <int D>
struct Sums {
    float ref, l;  // l: this lane's tokens only
    v4f o[D / 16];
    __device__ void clear() {
        ref = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int f = 0; f < D / 16; ++f) o[f] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
};

// Where a tile's tokens lie: every lane takes token lane % TILE.  peek asks
// the table, a tile ahead of its use; resolve makes a place of the answer,
// and a ballot over ok says which tokens are there.
struct Place {
    uint32_t unit;
    bool ok, stray;
};
template <int TILE>
__device__ __forceinline__ uint32_t peek(const PagedPool& p, const int32_t* table, uint32_t tokens, int tile, int lane) {
    return (uint32_t)table[p.page_tokens.quotient(min((uint32_t)tile * TILE + (lane & (TILE - 1)), tokens - 1))];
}
template <int TILE>
__device__ __forceinline__ Place resolve(const PagedPool& p, uint32_t page, uint32_t tokens, int tile, int lane) {
    const uint32_t t = (uint32_t)tile * TILE + (lane & (TILE - 1));
    Place at;
    at.stray = page >= p.pages;
    at.ok = t < tokens && !at.stray;
    at.unit = at.ok ? page * p.page_units + (t - p.page_tokens.quotient(t) * p.page_tokens.d) * p.slot_units : 0;
    return at;
}

// A tile's weights as operands of the second product.
template <bool IO, bool KV, int D>
struct Weights {
    static constexpr int kParts = Form<IO, KV, D>::kWeightParts, kMine = Form<IO, KV, D>::kMine;
    v4u part[kParts];  // of bfloat16; a 32-bit cache takes the weights as they are
    __device__ void operator=(const float (&w)[kMine]) {
        if constexpr (!KV) {
            part[0] = v4u{__float_as_uint(w[0]), __float_as_uint(w[1]), __float_as_uint(w[2]), __float_as_uint(w[3])};
        } else {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = w[j];
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
#pragma unroll
                for (int j = 0; j < 4; ++j) part[p][j] = pack_high(x[2 * j], x[2 * j + 1]);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] -= high_part(x[j]);
            }
        }
    }
};

// A tile's weights e^(s - m) from its scores, m the query's reference: the
// sums are brought to a new one only when a score passes the old one by
// 2^kRaise, which 32-bit sums hold with ease (64 rows over 32768 tokens 64 us;
// with every higher score 69).
template <bool IO, bool KV, int D>
__device__ __forceinline__ void weigh(const v4f (&sc)[Form<IO, KV, D>::kHalves], uint32_t there, float to_log2,
                                      int quarter, Sums<D>& s, Weights<IO, KV, D>& weights) {
    constexpr int N = Form<IO, KV, D>::kMine;
    float w[N];
    constexpr uint32_t kAll = N == 8 ? 0xffffffffu : 0xffffu;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        w[j] = Form<IO, KV, D>::kScaled ? sc[j >> 2][j & 3] : sc[j >> 2][j & 3] * to_log2;
        if (there != kAll && !(there >> (16 * (j >> 2) + 4 * quarter + (j & 3)) & 1u)) w[j] = -INFINITY;
        top = fmaxf(top, w[j]);
    }
    top = fmaxf(top, other_quarter<16>(top));
    top = fmaxf(top, other_quarter<32>(top));
    if (__any(top > s.ref + kRaise)) {
        const float to = fmaxf(top, s.ref);
        const float keep = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(s.ref - to);
        s.ref = to;
        s.l *= keep;
#pragma unroll
        for (int f = 0; f < D / 16; ++f) s.o[f] *= keep;
    }
    const float sub = s.ref == -INFINITY ? 0.0f : s.ref;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        w[j] = __builtin_amdgcn_exp2f(w[j] - sub);
        s.l += w[j];
    }
    weights = w;
}

// Values of tokens that are not there weigh 0, and may be anything.
template <bool KV, int N, int VR>
__device__ __forceinline__ void drop_values(uint32_t (&v)[N][VR], uint32_t there, int quarter) {
    if (there == (N == 8 ? 0xffffffffu : 0xffffu)) return;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t keep = (there >> (16 * (j >> 2) + 4 * quarter + (j & 3)) & 1u) ? 0xffffffffu : 0u;
#pragma unroll
        for (int x = 0; x < VR; ++x) v[j][x] &= keep;
    }
}

// One load's worth of a tile's value rows, weighted, added to the sums.
template <bool IO, bool KV, int D, int N, int VR>
__device__ __forceinline__ void add_values(const uint32_t (&v)[N][VR], const Weights<IO, KV, D>& w, int g, Sums<D>& s) {
    using F = Form<IO, KV, D>;
    constexpr int W = F::kWide;
    if constexpr (KV) {
        // two accumulators at a time: a product waits for the one before it on
        // the same accumulator (four would not leave the registers for it)
#pragma unroll
        for (int from = 0; from < W; from += 2) {
            v4u rows[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    rows[i][j] = __builtin_amdgcn_perm(v[2 * j + 1][(from + i) >> 1], v[2 * j][(from + i) >> 1],
                                                       i & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int p = 0; p < F::kWeightParts; ++p)
#pragma unroll
                for (int i = 0; i < 2; ++i) s.o[g * W + from + i] = mfma_bf16(rows[i], w.part[p], s.o[g * W + from + i]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int i = 0; i < W; ++i)
                s.o[g * W + i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[j][i]),
                                                                      __uint_as_float(w.part[0][j]), s.o[g * W + i], 0, 0, 0);
    }
}

// Tiles tile, tile + step, ... before `end` of one table added to the sums;
// page is what the table says of the first.  Bound by memory where the tiles
// are read once (5.3 TB/s of a bfloat16 cache, 5.6 of a 32-bit one), by the
// chain of a tile's loads and products where a wave has few: one row of 2048
// tokens, a tile to a wave, 7.6 us.
template <bool IO, bool KV, int D>
__device__ __forceinline__ void add_tiles(const PagedAttnArgs& a, const v4u* queries, int n, const int32_t* table,
                                          uint32_t tokens, int tile, int end, int step, int kvh, uint32_t page,
                                          Sums<D>& s, int& bad) {
    using F = Form<IO, KV, D>;
    constexpr int W = F::kWide, H = F::kHalves, N = F::kMine;
    constexpr int ES = KV ? 2 : 4, VR = W * ES / 4;  // registers of a value row per load
    const int lane = threadIdx.x & 63, quarter = lane >> 4, col = lane & 15;
    const float to_log2 = F::kScaled ? 1.0f : a.scale * kLog2e;
    const char* const keys = (const char*)a.pool.keys;
    const char* const values = (const char*)a.pool.values;
    constexpr uint32_t kAll = H == 2 ? 0xffffffffu : 0xffffu;
    for (; tile < end; tile += step) {
        const Place at = resolve<F::kTile>(a.pool, page, tokens, tile, lane);
        if (at.stray) bad |= ZG_STATUS_PAGE;
        const uint32_t there = (uint32_t)__ballot(at.ok) & kAll;
        v4u k[H][F::kSteps];
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const char* row = keys + ((uint64_t)(uint32_t)__shfl((int)at.unit, 16 * h + col) * 64 + (uint32_t)kvh * D) * ES +
                              16 * quarter;
#pragma unroll
            for (int i = 0; i < F::kSteps; ++i) k[h][i] = *(const v4u*)(row + 64 * i);
        }
        // values: half of them now, half into the keys' registers once those
        // are used up, so that a lane needs at most 256
        uint32_t v[F::kLoads][N][VR];
        const char* vrow[N];
#pragma unroll
        for (int j = 0; j < N; ++j)
            vrow[j] = values + ((uint64_t)(uint32_t)__shfl((int)at.unit, 16 * (j >> 2) + 4 * quarter + (j & 3)) * 64 +
                                (uint32_t)kvh * D + W * col) * ES;
        auto load_values = [&](int g) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if constexpr (VR == 4) {
                    const v4u w = *(const v4u*)(vrow[j] + 16 * W * g * ES);
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[g][j][x] = w[x];
                } else {
                    const uint2 w = *(const uint2*)(vrow[j] + 16 * W * g * ES);
                    v[g][j][0] = w.x;
                    v[g][j][1] = w.y;
                }
            }
        };
        constexpr int kFirst = (F::kLoads + 1) / 2;
#pragma unroll
        for (int g = 0; g < kFirst; ++g) load_values(g);
        page = peek<F::kTile>(a.pool, table, tokens, tile + step, lane);
        __builtin_amdgcn_sched_barrier(0);
        // scores
        v4f sc[H];
#pragma unroll
        for (int h = 0; h < H; ++h) sc[h] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        // the queries' places are stepped through: kept for all steps they
        // would take the registers of a quarter of the keys
        int place = quarter * n + min(col, n - 1);
        asm volatile("" : "+v"(place));
#pragma unroll
        for (int i = 0; i < F::kSteps; ++i) {
#pragma unroll
            for (int p = 0; p < F::kParts; ++p, place += 4 * n) {
                const v4u b = queries[place];
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    if constexpr (KV) {
                        sc[h] = mfma_bf16(k[h][i], b, sc[h]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            sc[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[h][i][e]), __uint_as_float(b[e]),
                                                                         sc[h], 0, 0, 0);
                    }
                }
            }
            // two steps' queries in registers at a time
            if (i & 1) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int g = kFirst; g < F::kLoads; ++g) load_values(g);
        __builtin_amdgcn_sched_barrier(0);
        Weights<IO, KV, D> w;
        weigh<IO, KV, D>(sc, there, to_log2, quarter, s, w);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int g = 0; g < F::kLoads; ++g) {
            drop_values<KV>(v[g], there, quarter);
            add_values<IO, KV, D>(v[g], w, g, s);
        }
    }
}

// One triple per query: m and l side by side; the elements of `across`
// queries together in the order of the sums, 16 bytes per (accumulator,
// quarter, query), so that a wave stores whole lines.
template <int D>
__device__ __forceinline__ void store_sums(float2* stats, float* o, int across, int query, const v4f (&from)[D / 16],
                                           float ref, float l, int quarter) {
    if (quarter == 0) stats[query] = make_float2(ref, l);
    int at = (quarter * across + query) * 4;  // formed here, not held through the tiles
    asm volatile("" : "+v"(at));
#pragma unroll
    for (int f = 0; f < D / 16; ++f) *(v4f*)(o + f * 16 * across + at) = from[f];
}

// The sums of waves 0 .. n - 1 brought together in wave 0, in a fixed order;
// every wave of the workgroup calls this.
template <int D>
__device__ __forceinline__ void gather_waves(Sums<D>& s, int n, int wave, int lane, char* lds) {
    const int quarter = lane >> 4, col = lane & 15;
    float2* stats = (float2*)lds;  // [n][16]
    v4f* part = (v4f*)(lds + n * 16 * sizeof(float2));
    s.l += __shfl_xor(s.l, 16, kWave);
    s.l += __shfl_xor(s.l, 32, kWave);
    if (wave < n && quarter == 0) stats[wave * 16 + col] = make_float2(s.ref, s.l);
    __syncthreads();
    float top = -INFINITY;
    for (int w = 0; w < n; ++w) top = fmaxf(top, stats[w * 16 + col].x);
    const float sub = top == -INFINITY ? 0.0f : top;
    s.l = 0.0f;
    for (int w = 0; w < n; ++w) {
        const float2 x = stats[w * 16 + col];
        s.l += x.y * __builtin_amdgcn_exp2f(x.x == top ? 0.0f : x.x - sub);
    }
    const float keep = __builtin_amdgcn_exp2f(s.ref == top ? 0.0f : s.ref - sub);
    s.ref = top;
#pragma unroll
    for (int f = 0; f < D / 16; ++f) s.o[f] *= keep;
    while (n > 1) {
        const int half = (n + 1) / 2;
        if (wave >= half && wave < n)
#pragma unroll
            for (int f = 0; f < D / 16; ++f) part[((wave - half) * (D / 16) + f) * 64 + lane] = s.o[f];
        __syncthreads();
        if (wave < n - half)
#pragma unroll
            for (int f = 0; f < D / 16; ++f) s.o[f] += part[(wave * (D / 16) + f) * 64 + lane];
        __syncthreads();
        n = half;
    }
}
constexpr size_t gather_bytes(int waves, int head_dim) {
    return (size_t)waves * 16 * sizeof(float2) + (size_t)(waves / 2) * head_dim * 64;
}

// How a call is cut.  The prefix: `chunks` pieces of chunk_tiles tiles, each
// for `blocks` blocks of `block` queries and every kv head.  The rows' own
// tiles, in the order (row, kv head, tile), go in runs of `run` successive
// ones to the waves, `active` waves of each of the `groups` workgroups,
// whatever rows they belong to, so that long and short rows fill the card
// alike.  Where a workgroup's runs lie within one (row, kv head) its waves'
// sums are gathered to one piece; else each wave leaves a piece for each (row,
// kv head) that it meets.
struct Cut {
    int prefix_tiles, chunk_tiles, chunks, block, blocks, groups, per_group;  // per_group: most waves of a workgroup
    struct Run* runs;
    float2 *prefix_stats, *own_stats;
    float *prefix_o, *own_o;
};
// The pieces of one (row, kv head), by the waves that leave them: heads of
// successive waves, then mids of every `active`-th (gathered workgroups), then
// tails of successive waves.
struct Run {
    uint32_t head, heads, mid, mids, tail, tails, active;
};
struct Shares {
    uint32_t active, run, total;
};
__host__ __device__ inline Shares shares_of(uint32_t total, uint32_t groups, uint32_t per_group) {
    Shares s;
    const uint32_t each = (total + groups - 1) / groups;
    s.active = each < 1 ? 1 : each < per_group ? each : per_group;
    s.run = (total + groups * s.active - 1) / (groups * s.active);
    s.total = total;
    return s;
}
__device__ __forceinline__ Run run_of(const Shares& s, uint32_t from, uint32_t to) {
    Run r{0, 0, 0, 0, 0, 0, s.active};
    if (from == to) return r;
    const uint32_t whole = s.active * s.run, g0 = (from + whole - 1) / whole;
    const uint32_t g1 = to == s.total ? (to + whole - 1) / whole : to / whole;
    r.head = from / s.run;
    if (g0 >= g1) {
        r.heads = (to - 1) / s.run - r.head + 1;
        return r;
    }
    if (from < g0 * whole) r.heads = g0 * s.active - r.head;
    r.mid = g0 * s.active;
    r.mids = g1 - g0;
    r.tail = g1 * s.active;
    if (to > g1 * whole) r.tails = (to - 1) / s.run - r.tail + 1;
    return r;
}

__device__ __forceinline__ uint32_t own_tokens(const PagedAttnArgs& a, uint32_t r) {
    const int n = a.lengths[r];
    return n < 0 ? 0 : min((uint32_t)n, a.stride * a.pool.page_tokens.d);
}
// A query's triple of one piece of the prefix; the pieces lie like the rows'
// own, one after the other for all rows.
template <int D>
__device__ __forceinline__ void store_prefix(const PagedAttnArgs& a, const Cut& c, int piece, int query,
                                             const v4f (&from)[D / 16], float ref, float l, int quarter) {
    const int row = query / a.group;
    if (row >= (int)a.rows) return;
    const size_t at = ((size_t)piece * a.rows + row) * a.group;
    store_sums<D>(c.prefix_stats + at, c.prefix_o + at * D, a.group, query - row * a.group, from, ref, l, quarter);
}

// The piece of the prefix that a workgroup takes.  Workgroups id, id + 8, id +
// 16, ... run on one XCD: they are given the blocks of one piece, which that
// L2 then reads from memory once.
struct PieceOf {
    int block, kvh, chunk;
};
__device__ __forceinline__ PieceOf piece_of(const Cut& c, int kv_heads, int id) {
    const int pieces = c.chunks * kv_heads, whole = pieces / 8 * 8 * c.blocks;
    PieceOf p;
    int piece;
    if (id < whole) {
        p.block = id / 8 % c.blocks;
        piece = id / (8 * c.blocks) * 8 + id % 8;
    } else {
        p.block = (id - whole) % c.blocks;
        piece = (id - whole) / c.blocks + pieces / 8 * 8;
    }
    p.kvh = piece % kv_heads;
    p.chunk = piece / kv_heads;
    return p;
}

template <bool IO, bool KV, int D>
__device__ __forceinline__ void prefix_block(const PagedAttnArgs& a, const Cut& c, int id, char* lds) {
    const int tid = threadIdx.x, lane = tid & 63, quarter = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const PieceOf at_piece = piece_of(c, a.pool.kv_heads, id);
    const int block = at_piece.block, kvh = at_piece.kvh, chunk = at_piece.chunk;
    const int queries = (int)a.rows * a.group;
    struct {
        const void* base;
        const PagedAttnArgs& a;
        int first, last, kvh;
        __device__ size_t operator()(int m) const {
            const int f = min(first + m, last), r = f / a.group;
            return r * a.q_stride + (size_t)(kvh * a.group + f - r * a.group) * D;
        }
    } who{a.q, a, block * 16, queries - 1, kvh};
    const int first = chunk * c.chunk_tiles;
    const uint32_t page = peek<Form<IO, KV, D>::kTile>(a.pool, a.prefix, a.prefix_tokens, first + wave, lane);
    stage_queries<IO, KV, D>((v4u*)lds, 16, tid, 256, a.scale * kLog2e, who);
    __syncthreads();
    Sums<D> s;
    s.clear();
    int bad = 0;
    add_tiles<IO, KV, D>(a, (const v4u*)lds, 16, a.prefix, a.prefix_tokens, first + wave,
                         min(first + c.chunk_tiles, c.prefix_tiles), 4, kvh, page, s, bad);
    if (bad && a.status) atomicOr(a.status, bad);
    __syncthreads();
    gather_waves<D>(s, 4, wave, lane, lds);
    if (wave) return;
    store_prefix<D>(a, c, kvh * c.chunks + chunk, block * 16 + col, s.o, s.ref, s.l, quarter);
}

// LDS of own_block's table: 68 words for each wave, or one for all of them.
__host__ __device__ inline size_t table_bytes(uint32_t rows, int waves) {
    return rows <= 64 ? (size_t)waves * 68 * 4 : ((size_t)(rows + 1 + waves) * 4 + 15) / 16 * 16;
}

template <bool IO, bool KV, int D, int WAVES>
__device__ __forceinline__ void own_block(const PagedAttnArgs& a, const Cut& c, int id, char* lds) {
    using F = Form<IO, KV, D>;
    const int tid = threadIdx.x, lane = tid & 63, quarter = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // ahead[r]: tiles of the rows before r, in LDS.  Up to 64 rows every wave
    // finds them for itself, a row a lane, without a barrier; beyond, thread t
    // sums rows [t * per, (t + 1) * per).
    uint32_t* ahead = (uint32_t*)lds + (a.rows <= 64 ? wave * 68 : 0);
    int bad = 0;
    auto tiles_of = [&](uint32_t r) {
        const int n = a.lengths[r];
        const uint32_t room = a.stride * a.pool.page_tokens.d;
        if (n > 0 && (uint32_t)n > room) bad |= ZG_STATUS_POSITION;
        return n < 0 ? 0u : (min((uint32_t)n, room) + F::kTile - 1) / F::kTile;
    };
    auto sum_upto = [&](uint32_t x) {  // of this lane and the ones before it
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t y = (uint32_t)__shfl_up((int)x, off, kWave);
            if (lane >= off) x += y;
        }
        return x;
    };
    uint32_t all;
    if (a.rows <= 64) {
        const uint32_t mine = (uint32_t)lane < a.rows ? tiles_of(lane) : 0, upto = sum_upto(mine);
        if ((uint32_t)lane < a.rows) ahead[lane] = upto - mine;
        all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
        if (lane == 0) ahead[a.rows] = all;
        same_wave();
    } else {
        uint32_t* sums = ahead + a.rows + 1;
        const uint32_t per = (a.rows + 64 * WAVES - 1) / (64 * WAVES), r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
        uint32_t mine = 0;
        for (uint32_t r = r0; r < r1; ++r) mine += tiles_of(r);
        const uint32_t upto = sum_upto(mine);
        if (lane == 63) sums[wave] = upto;
        __syncthreads();
        uint32_t at = upto - mine;
        for (int w = 0; w < wave; ++w) at += sums[w];
        for (uint32_t r = r0; r < r1; ++r) {
            ahead[r] = at;
            at += tiles_of(r);
        }
        all = 0;
        for (int w = 0; w < WAVES; ++w) all += sums[w];
        all = (uint32_t)__builtin_amdgcn_readfirstlane((int)all);
        if (tid == 0) ahead[a.rows] = all;
        __syncthreads();
    }
    if (bad && a.status && id == 0) atomicOr(a.status, bad);
    const uint32_t kvs = a.pool.kv_heads;
    const Shares share = shares_of(all * kvs, c.groups, c.per_group);
    if (id == c.groups - 1)  // for the join; the last workgroup has the least to do
        for (uint32_t i = tid; i < a.rows * kvs; i += 64 * WAVES) {
            const uint32_t r = i / kvs, n = ahead[r + 1] - ahead[r], from = ahead[r] * kvs + (i - r * kvs) * n;
            c.runs[i] = run_of(share, from, from + n);
        }
    const uint32_t w = id * share.active + wave, from = id * share.active * share.run;
    uint32_t t = min(w * share.run, share.total);
    const uint32_t end = (uint32_t)wave < share.active ? min(t + share.run, share.total) : t;
    if (from >= share.total) return;
    auto at_row = [&](uint32_t r) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)ahead[r]); };
    // the row that holds the workgroup's first tile: the last one with
    // ahead[row] * kvs <= from
    uint32_t r = 0;
    for (uint32_t lo = 0, hi = a.rows; hi - lo > 1;) {
        const uint32_t mid = (lo + hi) / 2;
        if (at_row(mid) * kvs <= from) lo = r = mid;
        else hi = mid;
    }
    // one (row, kv head) for the whole workgroup?
    const uint32_t in_first = from - at_row(r) * kvs, tiles = at_row(r + 1) - at_row(r);
    const uint32_t upto = min(from + share.active * share.run, share.total);
    const bool gathered = upto - from <= tiles - in_first % tiles;
    v4u* queries = (v4u*)(lds + table_bytes(a.rows, WAVES)) + wave * F::kParts * F::kSteps * 4 * a.group;
    bad = 0;
    Sums<D> s;
    s.clear();
    while (t < end) {
        const uint32_t before = at_row(r), n = at_row(r + 1) - before;
        if ((before + n) * kvs <= t) {
            ++r;
            continue;
        }
        const uint32_t in_row = t - before * kvs, kvh = in_row / n, tile = in_row - kvh * n;
        const uint32_t upto_tile = min(n, tile + (end - t));
        struct {
            const void* base;
            size_t first;
            __device__ size_t operator()(int m) const { return first + (size_t)m * D; }
        } who{a.q, r * a.q_stride + (size_t)kvh * a.group * D};
        const int32_t* const table = a.table + (size_t)r * a.stride;
        const uint32_t here = own_tokens(a, r), page = peek<F::kTile>(a.pool, table, here, (int)tile, lane);
        stage_queries<IO, KV, D>(queries, a.group, lane, 64, a.scale * kLog2e, who);
        same_wave();
        add_tiles<IO, KV, D>(a, queries, a.group, table, here, (int)tile, (int)upto_tile, 1, (int)kvh, page, s, bad);
        same_wave();
        t += upto_tile - tile;
        if (gathered) break;
        s.l += __shfl_xor(s.l, 16, kWave);
        s.l += __shfl_xor(s.l, 32, kWave);
        const size_t piece = (size_t)w + r * kvs + kvh;
        if (col < a.group)
            store_sums<D>(c.own_stats + piece * a.group, c.own_o + piece * a.group * D, a.group, col, s.o, s.ref,
                          s.l, quarter);
        s.clear();
    }
    if (bad && a.status) atomicOr(a.status, bad);
    if (!gathered) return;
    __syncthreads();
    gather_waves<D>(s, share.active, wave, lane, lds);
    const size_t piece = (size_t)w + r * kvs + in_first / tiles;
    if (wave == 0 && col < a.group)
        store_sums<D>(c.own_stats + piece * a.group, c.own_o + piece * a.group * D, a.group, col, s.o, s.ref, s.l,
                      quarter);
}

// Over the prefix 16 queries a workgroup, whose four waves take tiles of their
// own, straight into registers.
template <bool IO, bool KV, int D>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(PagedAttnArgs a, Cut c) {
    extern __shared__ __align__(16) char lds[];
    const int over_prefix = c.chunks * c.blocks * a.pool.kv_heads;
    if ((int)blockIdx.x < over_prefix) prefix_block<IO, KV, D>(a, c, blockIdx.x, lds);
    else own_block<IO, KV, D, 4>(a, c, blockIdx.x - over_prefix, lds);
}

constexpr int kManyWaves = 8, kManyQueries = 16 * kManyWaves;
constexpr int kBuffers = 4;                         // tiles in LDS: two in use, two coming
constexpr int kSegment = 64;                        // tiles looked up at a time

// Many queries over the prefix: each of eight waves holds 16 queries and their
// sums in registers, and all go through the same tiles, which are copied
// straight to LDS, two in use and two coming; a tile is read from memory once
// for 128 queries.  In LDS the 16-byte pieces of row t are exchanged by an xor of
// t, so that 16 lanes reading one piece of 16 rows meet 16 different banks.
// Bound by the matrix cores and what stands between their products: 64 rows
// over 32768 tokens (256-element heads) 64 us, 52 GFLOP of three-part bfloat16
// products = 0.8 PFLOP/s where a large library product reaches 1.1, with 16-bit
// queries 49 us; with own tokens 91 MB are fetched of 88 there are.  Of a pair
// of tiles the scores take 1800 cycles (1536 of them products), the values 2420
// (1536, and 64 byte permutations that transpose them), weights and copies the
// rest.  16 queries and their sums fill a wave's registers, so a SIMD holds two
// waves; copies placed elsewhere between the products, another priority in
// them, or half the waves a phase later took as long or longer.
template <bool IO, bool KV, int D>
__device__ __forceinline__ void many_block(const PagedAttnArgs& a, const Cut& c, int id, char* lds) {
    using F = Form<IO, KV, D>;
    constexpr int W = F::kWide, H = F::kHalves, N = F::kMine;
    constexpr int ES = KV ? 2 : 4, VR = W * ES / 4;
    constexpr int kRow = D * ES, kPieces = kRow / 16;   // bytes and 16-byte pieces of a row
    constexpr int kHalf = F::kTile * kRow;              // bytes of a tile's keys; its values follow
    constexpr int kCopies = 2 * kHalf / 1024 / kManyWaves;  // 1 KB each, of a wave
    constexpr uint32_t kAll = H == 2 ? 0xffffffffu : 0xffffu;
    const int lane = threadIdx.x & 63, quarter = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float to_log2 = F::kScaled ? 1.0f : a.scale * kLog2e;
    const PieceOf at_piece = piece_of(c, a.pool.kv_heads, id);
    const int kvh = at_piece.kvh, queries = (int)a.rows * a.group;
    const int first = at_piece.chunk * c.chunk_tiles, end = min(first + c.chunk_tiles, c.prefix_tiles);
    auto swizzle = [](int row) { return kPieces >= 16 ? row & 15 : row >> 1 & 7; };
    // where this lane reads: its first piece of a key row and of a value row;
    // step i of a key is the piece xor 4 i, value row j the piece xor j
    int key_at = col * kRow + 16 * (quarter ^ swizzle(col));
    int value_at = kHalf + 4 * quarter * kRow +
                   (VR == 4 ? 16 * (col ^ swizzle(4 * quarter)) : 16 * ((col >> 1) ^ swizzle(4 * quarter)) + 8 * (col & 1));

    // the wave's queries: asked for first, used last
    const int mine = at_piece.block * kManyQueries + 16 * wave + col, f = min(mine, queries - 1), r = f / a.group;
    const size_t from = r * a.q_stride + (size_t)(kvh * a.group + f - r * a.group) * D;
    const bool live = at_piece.block * kManyQueries + 16 * wave < queries;
    v4u raw[F::kSteps][KV && !IO ? 2 : 1];
#pragma unroll
    for (int i = 0; i < F::kSteps; ++i) {
        if constexpr (!KV) {
            raw[i][0] = __builtin_bit_cast(v4u, load4<IO>(a.q, from + 16 * i + 4 * quarter));
        } else if constexpr (IO) {
            raw[i][0] = *(const v4u*)((const uint16_t*)a.q + from + 32 * i + 8 * quarter);
        } else {
            raw[i][0] = *(const v4u*)((const float*)a.q + from + 32 * i + 8 * quarter);
            raw[i][1] = *(const v4u*)((const float*)a.q + from + 32 * i + 8 * quarter + 4);
        }
    }

    // the places of a segment's tokens, looked up once for the workgroup; all
    // ones: the token is not there
    uint32_t* const units = (uint32_t*)(lds + kBuffers * 2 * kHalf);
    // Addresses are formed anew for each tile (the empty asm keeps them from
    // being held): registers are short, and a spilled one, reloaded, would
    // wait for the copies under way.
    auto copy = [&](int local, int buffer) {
        int self = lane;
        asm volatile("" : "+v"(self));
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const int x = wave * kCopies + i, within = (x * 1024 & (kHalf - 1)) / 16 + self;
            const int row = within / kPieces, piece = within % kPieces ^ swizzle(row);
            const uint32_t unit = units[local * F::kTile + row];
            const char* from = (const char*)(x * 1024 < kHalf ? a.pool.keys : a.pool.values) +
                               ((uint64_t)(unit == ~0u ? 0u : unit) * 64 + (uint32_t)kvh * D) * ES + 16 * piece;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                             (__attribute__((address_space(3))) void*)(lds + buffer * 2 * kHalf + x * 1024),
                                             16, 0, 0);
        }
    };
    int bad = 0;
    auto look_up = [&](int from, int n) {
        for (int i = threadIdx.x; i < n * F::kTile; i += 64 * kManyWaves) {
            const uint32_t t = (uint32_t)from * F::kTile + i;
            uint32_t unit = ~0u;
            if (t < a.prefix_tokens) {
                const uint32_t pg = a.pool.page_tokens.quotient(t), page = (uint32_t)a.prefix[pg];
                if (page < a.pool.pages)
                    unit = page * a.pool.page_units + (t - pg * a.pool.page_tokens.d) * a.pool.slot_units;
                else
                    bad |= ZG_STATUS_PAGE;
            }
            units[i] = unit;
        }
    };
    // the copies of tiles `local` and the next, and which of their tokens are
    // there; past the segment's last tile that one again
    int held = min(kSegment, end - first);  // tiles of the segment in `units`
    uint32_t coming[2];
    auto fetch = [&](int local, int buffer) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int x = min(local + i, held - 1);
            coming[i] = (uint32_t)__ballot(units[x * F::kTile + (lane & (F::kTile - 1))] != ~0u) & kAll;
            copy(x, buffer + i);
        }
    };
    look_up(first, held);
    __syncthreads();
    fetch(0, 0);

    // the queries' parts, in operand order
    v4u q[F::kParts][F::kSteps];
#pragma unroll
    for (int i = 0; i < F::kSteps; ++i) {
        if constexpr (!KV) {
            q[0][i] = __builtin_bit_cast(v4u, __builtin_bit_cast(v4f, raw[i][0]) * (a.scale * kLog2e));
        } else if constexpr (IO) {
            q[0][i] = raw[i][0];
        } else {
            v4f x[2] = {__builtin_bit_cast(v4f, raw[i][0]) * (a.scale * kLog2e),
                        __builtin_bit_cast(v4f, raw[i][1]) * (a.scale * kLog2e)};
#pragma unroll
            for (int p = 0; p < F::kParts; ++p) {
#pragma unroll
                for (int j = 0; j < 4; ++j) q[p][i][j] = pack_high(x[j >> 1][(2 * j) & 3], x[j >> 1][(2 * j + 1) & 3]);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j >> 2][j & 3] -= high_part(x[j >> 2][j & 3]);
            }
        }
    }
    Sums<D> s;
    s.clear();
    Weights<IO, KV, D> w;
    uint32_t v[N][VR];
    auto load_values = [&](int g, int buffer) {
        const char* const data = lds + buffer * 2 * kHalf;
        if (g == 0) asm volatile("" : "+v"(value_at));
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int exchange = 16 * (kPieces >= 16 ? j & 3 : (j & 3) >> 1);
            const char* from = data + (value_at ^ exchange) + (16 * (j >> 2) + (j & 3)) * kRow + 256 * g;
            if constexpr (VR == 4) {
                const v4u x = *(const v4u*)from;
#pragma unroll
                for (int y = 0; y < 4; ++y) v[j][y] = x[y];
            } else {
                const uint2 x = *(const uint2*)from;
                v[j][0] = x.x;
                v[j][1] = x.y;
            }
        }
    };
    // a tile's values, the first load of them on its way already
    auto add = [&](uint32_t there, int buffer) {
#pragma unroll
        for (int g = 0; g < F::kLoads; ++g) {
            if (g) load_values(g, buffer);
            drop_values<KV>(v, there, quarter);
            add_values<IO, KV, D>(v, w, g, s);
        }
    };
    // Two tiles between barriers: within them the two waves of a SIMD drift
    // apart, so that one's products run beside the other's weights.
    for (int tile = first, local = 0; tile < end; tile += 2, local += 2) {
        if (local >= held) {
            // the next segment: everyone is done with this one, and the copies
            // past its end have landed
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            held = min(kSegment, end - tile);
            look_up(tile, held);
            __syncthreads();
            local = 0;
            fetch(0, (tile - first) & 2);
        }
        uint32_t there[2] = {coming[0], coming[1]};
        const int pair = (tile - first) & 2;  // its first buffer
        // both tiles' copies have landed; after the barrier everyone's have,
        // and the other two buffers have been read
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (!live) {
            fetch(local + 2, pair ^ 2);
            continue;
        }
#pragma unroll 1
        for (int half = 0; half < 2 && tile + half < end; ++half) {
        const int buffer = pair + half;
        const char* const data = lds + buffer * 2 * kHalf;
        asm volatile("" : "+v"(key_at));
        // the keys of two steps are on their way while a third is used
        v4u k[3][H];
        auto load_keys = [&](int i) {
#pragma unroll
            for (int h = 0; h < H; ++h)
                k[i % 3][h] = *(const v4u*)(data + (key_at ^ 64 * (i & 3)) + 16 * h * kRow + 256 * (i / 4));
        };
        load_keys(0);
        if (F::kSteps > 1) load_keys(1);
        v4f sc[H];
#pragma unroll
        for (int h = 0; h < H; ++h) sc[h] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < F::kSteps; ++i) {
            if (i + 2 < F::kSteps) load_keys(i + 2);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int p = 0; p < F::kParts; ++p)
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    if constexpr (KV) {
                        sc[h] = mfma_bf16(k[i % 3][h], q[p][i], sc[h]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            sc[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[i % 3][h][e]),
                                                                            __uint_as_float(q[0][i][e]), sc[h], 0, 0, 0);
                    }
                }
            __builtin_amdgcn_sched_barrier(0);
        }
        load_values(0, buffer);
        if (half == 0) fetch(local + 2, pair ^ 2);
        __builtin_amdgcn_sched_barrier(0);
        weigh<IO, KV, D>(sc, there[half], to_log2, quarter, s, w);
        add(there[half], buffer);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy outlives the workgroup's LDS
    if (bad && a.status) atomicOr(a.status, bad);
    s.l += __shfl_xor(s.l, 16, kWave);
    s.l += __shfl_xor(s.l, 32, kWave);
    store_prefix<D>(a, c, kvh * c.chunks + at_piece.chunk, mine, s.o, s.ref, s.l, quarter);
}

template <bool IO, bool KV, int D>
__global__ __launch_bounds__(64 * kManyWaves, 2) void paged_attn_many_kernel(PagedAttnArgs a, Cut c) {
    extern __shared__ __align__(16) char lds[];
    // One workgroup fits a CU: those that take a piece of the prefix are the
    // first, the rows' own tiles go to the last ones, and where they meet a
    // workgroup does one after the other.
    const int over_prefix = c.chunks * c.blocks * a.pool.kv_heads, own = (int)gridDim.x - 1 - (int)blockIdx.x;
    if ((int)blockIdx.x < over_prefix) {
        many_block<IO, KV, D>(a, c, blockIdx.x, lds);
        if (own >= c.groups) return;
        __syncthreads();
    }
    if (own < c.groups) own_block<IO, KV, D, kManyWaves>(a, c, own, lds);
}

// Workgroup (kv head, row, four accumulators): a thread owns 16 bytes of the
// pieces, (accumulator, quarter, query), and every n-th piece; the n threads
// of one item are joined at the end, in order.  Pieces lie in the order of the
// sums, so that neighbouring threads read whole lines: 64 rows, 64 pieces each
// for a head, 34 MB, take 10 us.  A few pieces are a launch, the look at `runs`
// and two rounds of loads: 4 to 5 us.
template <bool IO, int D, int W, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_join_kernel(PagedAttnArgs a, Cut c) {
    constexpr int kJoin = THREADS == 1024 ? 4 : 8;  // pieces that a thread has under way
    __shared__ v4f parts[THREADS];
    __shared__ float2 stats[THREADS];
    const uint32_t kvh = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
    const Run run = c.runs[r * a.pool.kv_heads + kvh];
    const uint32_t items = 16 * a.group, n = THREADS / items, item = tid % items, nth = tid / items;
    const uint32_t col = item % a.group, fq = blockIdx.z * 16 + item / a.group;
    const uint32_t chunks = c.chunks, pieces = chunks + run.heads + run.mids + run.tails;
    if (a.lengths[r] < 0) return;
    const size_t own_base = r * a.pool.kv_heads + kvh;
    float top = -INFINITY, l = 0.0f;
    v4f o = {};
    if (nth < n)
        for (uint32_t i = nth; i < pieces; i += kJoin * n) {
            v4f x[kJoin];
            float2 y[kJoin];
#pragma unroll
            for (int u = 0; u < kJoin; ++u) {
                // past the last piece: the last one, with no weight
                const uint32_t p = min(i + u * n, pieces - 1);
                uint32_t w = p - chunks;
                if (w < run.heads) w += run.head;
                else if (w < run.heads + run.mids) w = run.mid + (w - run.heads) * run.active;
                else w = run.tail + (w - run.heads - run.mids);
                const bool shared = p < chunks;
                const size_t at = (shared ? (size_t)(kvh * chunks + p) * a.rows + r : own_base + w) * a.group;
                y[u] = (shared ? c.prefix_stats : c.own_stats)[at + col];
                x[u] = *(const v4f*)((shared ? c.prefix_o : c.own_o) + at * D + (fq * a.group + col) * 4);
            }
            float to = top;
#pragma unroll
            for (int u = 0; u < kJoin; ++u) to = fmaxf(to, y[u].x);
            const float sub = to == -INFINITY ? 0.0f : to;
            const float keep = __builtin_amdgcn_exp2f(top == to ? 0.0f : top - sub);
            l *= keep;
            o *= keep;
            top = to;
#pragma unroll
            for (int u = 0; u < kJoin; ++u)
                if (i + u * n < pieces) {
                    const float e = __builtin_amdgcn_exp2f(y[u].x == to ? 0.0f : y[u].x - sub);
                    l += e * y[u].y;
                    o += e * x[u];
                }
        }
    parts[tid] = o;
    stats[tid] = make_float2(top, l);
    __syncthreads();
    if (tid < items) {
        float to = top;
#pragma unroll 4
        for (uint32_t i = 1; i < n; ++i) to = fmaxf(to, stats[tid + i * items].x);
        const float sub = to == -INFINITY ? 0.0f : to;
        const float keep = __builtin_amdgcn_exp2f(top == to ? 0.0f : top - sub);
        l *= keep;
        o *= keep;
#pragma unroll 4
        for (uint32_t i = 1; i < n; ++i) {
            const float2 y = stats[tid + i * items];
            const float e = __builtin_amdgcn_exp2f(y.x == to ? 0.0f : y.x - sub);
            l += e * y.y;
            o += e * parts[tid + i * items];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = l == 0.0f ? 0.0f : o[j] / l;
    }
    __syncthreads();
    if (tid < items) parts[tid] = o;
    __syncthreads();
    // accumulators 4 z .. 4 z + 3 are four successive elements: thread (query,
    // quarter, register) stores them
    if (tid >= items) return;
    const uint32_t head = tid / 16, quarter = tid / 4 % 4, reg = tid % 4, f = blockIdx.z * 4;
    v4f out;
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = parts[(j * 4 + quarter) * a.group + head][reg];
    store4<IO>(a.out, r * a.out_stride + (size_t)(kvh * a.group + head) * D + 16 * W * (f / W) + W * (4 * quarter + reg) + f % W,
               out);
}

// ------------------------------------------------------------------- host

// Queries of one kv head that go over a tile of the prefix together: 16, in one
// wave, or 128, in a workgroup that reads the tile for all of them.  The
// latter is slow to start and leaves larger pieces, so it takes over where 16
// at a time would give each of 1024 waves more than 6 tiles.  256-element heads,
// 8 queries a row on 2 kv heads, both launches, 16 at a time and 128: 32 rows
// over 512 tokens 13.5 and 17.9 us, over 2048 16.6 and 21.4, over 8192 (4 tiles
// a wave) 23.6 and 29.7, over 16384 (8) 35.0 and 35.5, over 32768 57.0 and 52.0;
// 16-bit queries there 21.9 and 24.8, 32.1 and 29.3, 51.9 and 42.0; 16 rows over
// 32768 (8) 36.2 and 39.4; 128-element heads, 64 rows over 2048 (5) 19.6 and
// 17.4, 32 over 8192 (10) 27.9 and 26.3.
constexpr uint64_t kFewTiles = 6 * 1024;
static int block_of(uint64_t queries, int kv_heads, uint64_t tiles) {
    return queries <= 16 || (queries + 15) / 16 * kv_heads * tiles <= kFewTiles ? 16 : kManyQueries;
}

// The workspace's parts; its bytes.
static size_t lay_out(Cut& c, size_t runs, size_t prefix_rows, size_t own_rows, int head_dim, void* workspace) {
    char* at = (char*)workspace;
    auto take = [&](size_t n) {
        char* p = at;
        at += (n + 255) / 256 * 256;
        return p;
    };
    c.runs = (Run*)take(runs * sizeof(Run));
    c.prefix_stats = (float2*)take(prefix_rows * sizeof(float2));
    c.own_stats = (float2*)take(own_rows * sizeof(float2));
    c.prefix_o = (float*)take(prefix_rows * head_dim * sizeof(float));
    c.own_o = (float*)take(own_rows * head_dim * sizeof(float));
    return (size_t)(at - (char*)workspace);
}

static Cut cut_of(uint32_t rows, int q_heads, int kv_heads, int head_dim, int tile, uint32_t prefix_tokens,
                  uint64_t row_tokens, size_t query_bytes, void* workspace) {
    Cut c{};
    const int group = q_heads / kv_heads;
    c.prefix_tiles = (int)((prefix_tokens + tile - 1) / tile);
    c.block = block_of((uint64_t)rows * group, kv_heads, c.prefix_tiles);
    c.blocks = (int)(((uint64_t)rows * group + c.block - 1) / c.block);
    if (c.prefix_tiles) {
        // More pieces run side by side, and each costs the join: with T tiles
        // in all, a tile taking some 2 us and a piece of 128 queries adding
        // 0.05 us (256-element heads), sqrt(40 T) pieces.  32 rows over 16384
        // tokens: 256 pieces 31 + 9 us, 172 pieces 28 + 8, 128 pieces 31 + 8,
        // 104 pieces 36 + 6.  A piece of few queries is cheap: one tile for each
        // wave, up to a piece to a CU (two: 32 rows over 8192 23 + 6, one 20 + 4).
        const int share = kv_heads * c.blocks;
        const int most = c.block == kManyQueries ? (int)std::sqrt(40.0 * c.prefix_tiles * share) / share
                                                 : std::min((c.prefix_tiles + 3) / 4, kCus / share);
        const int want = std::max(1, std::min({most, c.prefix_tiles, kCus / share}));
        c.chunk_tiles = (c.prefix_tiles + want - 1) / want;
        // many queries take tiles in pairs; one piece to a CU
        if (c.block == kManyQueries && c.chunk_tiles % 2) {
            const int less = std::max(2, c.chunk_tiles - 1);
            c.chunk_tiles = (c.prefix_tiles + less - 1) / less * share <= kCus ? less : c.chunk_tiles + 1;
        }
        c.chunks = (c.prefix_tiles + c.chunk_tiles - 1) / c.chunk_tiles;
    }
    // eight waves' queries may not fit the LDS (16 to a kv head, in three parts)
    const bool many = c.chunks && c.block == kManyQueries;
    c.per_group = many && kManyWaves * group * query_bytes <= kOwnLds ? kManyWaves : 4;
    const uint64_t own_tiles = (uint64_t)rows * kv_heads * ((row_tokens + tile - 1) / tile);
    int most = kOwnWaves / c.per_group;
    if (many) {
        // the CUs that the prefix leaves, if they are a quarter of them (32 rows
        // with 2048 tokens of their own over 16384: 32 us, spread over all 39)
        const int left = kCus - c.chunks * c.blocks * kv_heads;
        most = left >= kCus / 4 ? left : kCus;
    }
    c.groups = (int)std::min<uint64_t>(most, own_tiles);
    const size_t prefix_rows = (size_t)kv_heads * c.chunks * rows * group;
    const size_t own_rows = ((size_t)c.groups * c.per_group + (size_t)rows * kv_heads) * group;
    lay_out(c, (size_t)rows * kv_heads, prefix_rows, own_rows, head_dim, workspace);
    return c;
}

// No call with at most as many rows, tokens a row and prefix tokens takes more: a
// piece of the prefix goes to a CU, or there is one for each block; a call that
// takes 16 queries at a time has only such calls below it.
size_t paged_attn_workspace(uint32_t rows, int q_heads, int kv_heads, int head_dim, int bf16, uint32_t prefix_tokens,
                            uint64_t row_tokens) {
    const uint64_t tile = bf16 ? 32 : 16, group = q_heads / kv_heads, queries = rows * group;
    const uint64_t tiles = (prefix_tokens + tile - 1) / tile, all = (uint64_t)kv_heads * tiles * queries;
    const bool many = tiles && block_of(queries, kv_heads, tiles) == kManyQueries;
    auto pieces = [&](uint64_t block) {
        return std::min(all, block * std::max<uint64_t>(kCus, (queries + block - 1) / block * kv_heads));
    };
    const uint64_t prefix_rows = std::max(pieces(16), many ? pieces(kManyQueries) : 0);
    const uint64_t own_tiles = (uint64_t)rows * kv_heads * ((row_tokens + tile - 1) / tile);
    const uint64_t groups = std::min<uint64_t>(kCus, own_tiles);
    const uint64_t own_rows = (groups * (many ? kManyWaves : 4) + (uint64_t)rows * kv_heads) * group;
    Cut c{};
    return lay_out(c, (size_t)rows * kv_heads, prefix_rows, own_rows, head_dim, nullptr);
}

// A staged query: 16 bytes for each part, step and quarter.
template <bool IO, bool KV, int D>
constexpr size_t query_bytes() {
    return (size_t)Form<IO, KV, D>::kParts * Form<IO, KV, D>::kSteps * 4 * 16;
}

template <bool IO, bool KV, int D>
static hipError_t launch(const PagedAttnArgs& a, hipStream_t st) {
    const Cut c = cut_of(a.rows, a.q_heads, a.pool.kv_heads, D, Form<IO, KV, D>::kTile, a.prefix_tokens,
                         (uint64_t)a.stride * a.pool.page_tokens.d, query_bytes<IO, KV, D>(), a.workspace);
    using F = Form<IO, KV, D>;
    const bool many = c.chunks && c.block == kManyQueries;
    const int waves = many ? kManyWaves : 4;
    constexpr size_t query = query_bytes<IO, KV, D>();
    const size_t own = std::max(table_bytes(a.rows, waves) + c.per_group * a.group * query, gather_bytes(c.per_group, D));
    size_t prefix = 0;
    if (many) prefix = (size_t)kBuffers * 2 * F::kTile * D * (KV ? 2 : 4) + (size_t)kSegment * F::kTile * 4;
    else if (c.chunks) prefix = std::max(query * c.block, gather_bytes(4, D));
    const size_t lds = std::max(prefix, own);
    void (*kernel)(PagedAttnArgs, Cut) = many ? paged_attn_many_kernel<IO, KV, D> : paged_attn_kernel<IO, KV, D>;
    if (lds > 65536) {
        hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    const int over_prefix = c.chunks * c.blocks * a.pool.kv_heads;
    kernel<<<many ? std::max(over_prefix, kCus) : over_prefix + c.groups, 64 * waves, lds, st>>>(a, c);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // Few workgroups or many pieces: more threads, and fewer pieces for each.
    // One row of 32768 tokens (8 workgroups) 15.9 -> 8.9 us, of 2048 5.8 -> 4.8,
    // 8 rows over a prefix of 32768 (64) 10.6 -> 6.1, 32 rows over 131072 in
    // 128 pieces (256) 13.0 -> 8.9; with 22 pieces there 4.2 -> 6.4.
    const dim3 grid(a.pool.kv_heads, a.rows, D / 64);
    if ((size_t)grid.x * grid.y * grid.z <= 64 || c.chunks > 64) paged_join_kernel<IO, D, F::kWide, 1024><<<grid, 1024, 0, st>>>(a, c);
    else paged_join_kernel<IO, D, F::kWide, 256><<<grid, 256, 0, st>>>(a, c);
    return hipGetLastError();
}

hipError_t paged_attn(const PagedAttnArgs& a, hipStream_t st) {
    auto by_dim = [&](auto io, auto kv) {
        constexpr bool IO = decltype(io)::value, KV = decltype(kv)::value;
        switch (a.pool.head_dim) {
        case 64: return launch<IO, KV, 64>(a, st);
        case 128: return launch<IO, KV, 128>(a, st);
        default: return launch<IO, KV, 256>(a, st);
        }
    };
    if (a.io_bf16) return a.pool.bf16 ? by_dim(std::true_type{}, std::true_type{}) : by_dim(std::true_type{}, std::false_type{});
    return a.pool.bf16 ? by_dim(std::false_type{}, std::true_type{}) : by_dim(std::false_type{}, std::false_type{});
}

}  // namespace zg

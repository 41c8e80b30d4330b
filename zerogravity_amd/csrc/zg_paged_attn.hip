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
// So the tile needs neither LDS nor a barrier, and each key and value is read
// from memory once per 16 MT queries.
#include <algorithm>

#include "zg_paged.hpp"

namespace zg {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

constexpr int kOwnGroups = 256;     // workgroups over the rows' own tiles
constexpr int kPrefixGroups = 256;  // about so many over the prefix
constexpr float kRaise = 8.0f;      // log2: how far a score may pass the reference before sums are rescaled

template <bool IO, bool KV, int D>
struct Form {
    // a 32-bit query enters a bfloat16 product as three parts of 8 bits, its
    // 24 in all; so do the weights of 32-bit outputs.  16-bit outputs take two
    // parts of a weight: 2^-16 of it is left out, a 256th of the output's
    // own rounding.
    static constexpr int kParts = KV ? (IO ? 1 : 3) : 1;
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

// Queries in LDS in operand order, 16 bytes per (part, step, quarter, query):
// a wave's read is contiguous.  `who` gives query m's elements in memory.
template <bool IO, bool KV, int D, typename Who>
__device__ __forceinline__ void stage_queries(v4u* lds, int n, int thread, int threads, Who who) {
    using F = Form<IO, KV, D>;
    constexpr int E = KV ? 8 : 4;
    for (int i = thread; i < n * (D / E); i += threads) {
        const int m = i % n, c = i / n;
        const size_t at = who(m) + c * E;
        if constexpr (!KV) {
            lds[c * n + m] = __builtin_bit_cast(v4u, load4<IO>(who.base, at));
        } else if constexpr (IO) {
            lds[c * n + m] = *(const v4u*)((const uint16_t*)who.base + at);
        } else {
            v4f x[2] = {load4<false>(who.base, at), load4<false>(who.base, at + 4)};
#pragma unroll
            for (int p = 0; p < F::kParts; ++p) {
                v4u w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = pack_high(x[j >> 1][(2 * j) & 3], x[j >> 1][(2 * j + 1) & 3]);
                lds[(p * (D / E) + c) * n + m] = w;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j >> 2][j & 3] -= high_part(x[j >> 2][j & 3]);
            }
        }
    }
}

// A wave's running sums for 16 MT queries: lane l holds query l % 16 of each
// tile; o[..][f][r] is element 16 W g + W (4 quarter + r) + i of it, f = W g + i.
template <int D, int MT>
struct Sums {
    float ref[MT], l[MT];  // l: this lane's tokens only
    v4f o[MT][D / 16];
    __device__ void clear() {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            ref[m] = -INFINITY;
            l[m] = 0.0f;
#pragma unroll
            for (int f = 0; f < D / 16; ++f) o[m][f] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
};

// Where a tile's tokens lie: every lane finds token lane % TILE, and a ballot
// says which are there.
struct Place {
    uint32_t unit;
    bool ok, stray;
};
template <int TILE>
__device__ __forceinline__ Place find(const PagedPool& p, const int32_t* table, uint32_t tokens, int tile, int lane) {
    const uint32_t t = (uint32_t)tile * TILE + (lane & (TILE - 1));
    const uint32_t pg = p.page_tokens.quotient(min(t, tokens - 1));
    const uint32_t page = (uint32_t)table[pg];
    Place at;
    at.stray = page >= p.pages;
    at.ok = t < tokens && !at.stray;
    at.unit = at.ok ? page * p.page_units + (t - pg * p.page_tokens.d) * p.slot_units : 0;
    return at;
}

// Tiles tile, tile + step, ... before `end` of one table added to the sums.
template <bool IO, bool KV, int D, int MT>
__device__ __forceinline__ void add_tiles(const PagedAttnArgs& a, const v4u* queries, int n, const int32_t* table,
                                          uint32_t tokens, int tile, int end, int step, int kvh, Sums<D, MT>& s,
                                          int& bad) {
    using F = Form<IO, KV, D>;
    constexpr int W = F::kWide, H = F::kHalves, N = F::kMine;
    constexpr int ES = KV ? 2 : 4, VR = W * ES / 4;  // registers of a value row per load
    const int lane = threadIdx.x & 63, quarter = lane >> 4, col = lane & 15;
    const float to_log2 = a.scale * 1.44269504088896341f;
    const char* const keys = (const char*)a.pool.keys;
    const char* const values = (const char*)a.pool.values;
    constexpr uint32_t kAll = H == 2 ? 0xffffffffu : 0xffffu;
    if (tile >= end) return;
    Place at = find<F::kTile>(a.pool, table, tokens, tile, lane);
    for (; tile < end; tile += step) {
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
        uint32_t v[N][F::kLoads][VR];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const char* row = values + ((uint64_t)(uint32_t)__shfl((int)at.unit, 16 * (j >> 2) + 4 * quarter + (j & 3)) * 64 +
                                        (uint32_t)kvh * D + W * col) * ES;
#pragma unroll
            for (int g = 0; g < F::kLoads; ++g) {
                if constexpr (VR == 4) {
                    const v4u w = *(const v4u*)(row + 16 * W * g * ES);
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[j][g][x] = w[x];
                } else {
                    const uint2 w = *(const uint2*)(row + 16 * W * g * ES);
                    v[j][g][0] = w.x;
                    v[j][g][1] = w.y;
                }
            }
        }
        if (tile + step < end) at = find<F::kTile>(a.pool, table, tokens, tile + step, lane);
        __builtin_amdgcn_sched_barrier(0);
        // scores
        v4f sc[MT][H];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < H; ++h) sc[m][h] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < F::kSteps; ++i) {
#pragma unroll
            for (int p = 0; p < F::kParts; ++p)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const int q = MT == 1 ? min(col, n - 1) : 16 * m + col;
                    const v4u b = queries[((p * F::kSteps + i) * 4 + quarter) * n + q];
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        if constexpr (KV) {
                            sc[m][h] = mfma_bf16(k[h][i], b, sc[m][h]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                sc[m][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                    __uint_as_float(k[h][i][e]), __uint_as_float(b[e]), sc[m][h], 0, 0, 0);
                        }
                    }
                }
            // two steps' queries in registers at a time
            if (i & 1) __builtin_amdgcn_sched_barrier(0);
        }
        // weights
        float w[MT][N];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                w[m][j] = sc[m][j >> 2][j & 3] * to_log2;
                if (there != kAll && !(there >> (16 * (j >> 2) + 4 * quarter + (j & 3)) & 1u)) w[m][j] = -INFINITY;
                top = fmaxf(top, w[m][j]);
            }
            top = fmaxf(top, __shfl_xor(top, 16, kWave));
            top = fmaxf(top, __shfl_xor(top, 32, kWave));
            if (__any(top > s.ref[m] + kRaise)) {
                const float to = fmaxf(top, s.ref[m]);
                const float keep = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(s.ref[m] - to);
                s.ref[m] = to;
                s.l[m] *= keep;
#pragma unroll
                for (int f = 0; f < F::kFrags; ++f) s.o[m][f] *= keep;
            }
            const float sub = s.ref[m] == -INFINITY ? 0.0f : s.ref[m];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                w[m][j] = __builtin_amdgcn_exp2f(w[m][j] - sub);
                s.l[m] += w[m][j];
            }
        }
        // values of tokens that are not there weigh 0, and may be anything
        if (there != kAll) {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (!(there >> (16 * (j >> 2) + 4 * quarter + (j & 3)) & 1u))
#pragma unroll
                    for (int g = 0; g < F::kLoads; ++g)
#pragma unroll
                        for (int x = 0; x < VR; ++x) v[j][g][x] = 0;
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (KV) {
            v4u part[MT][F::kWeightParts];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int p = 0; p < F::kWeightParts; ++p) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) part[m][p][j] = pack_high(w[m][2 * j], w[m][2 * j + 1]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[m][j] -= high_part(w[m][j]);
                }
#pragma unroll
            for (int g = 0; g < F::kLoads; ++g)
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    v4u rows;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        rows[j] = __builtin_amdgcn_perm(v[2 * j + 1][g][i >> 1], v[2 * j][g][i >> 1],
                                                        i & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                    for (int p = 0; p < F::kWeightParts; ++p)
#pragma unroll
                        for (int m = 0; m < MT; ++m)
                            s.o[m][g * W + i] = mfma_bf16(rows, part[m][p], s.o[m][g * W + i]);
                }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
#pragma unroll
                for (int g = 0; g < F::kLoads; ++g)
#pragma unroll
                    for (int i = 0; i < W; ++i)
#pragma unroll
                        for (int m = 0; m < MT; ++m)
                            s.o[m][g * W + i] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                __uint_as_float(v[j][g][i]), w[m][j], s.o[m][g * W + i], 0, 0, 0);
        }
    }
}

// One triple per query: m and l side by side, then the D elements.
template <int W, int D>
__device__ __forceinline__ void store_sums(float2* stats, float* o, size_t at, const v4f (&from)[D / 16], float ref,
                                           float l, int quarter) {
    if (quarter == 0) stats[at] = make_float2(ref, l);
#pragma unroll
    for (int g = 0; g < D / (16 * W); ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int x = 0; x < W; x += 4)
                *(v4f*)(o + at * D + 16 * W * g + W * (4 * quarter + r) + x) =
                    v4f{from[g * W + x][r], from[g * W + x + 1][r], from[g * W + x + 2][r], from[g * W + x + 3][r]};
}

// How a call is cut.  The prefix: `chunks` pieces of chunk_tiles tiles, each
// for `blocks` blocks of 16 MT queries and every kv head.  The rows' own
// tiles, in the order (row, kv head, tile): wave w of the `waves` takes c
// successive ones, c = ceil(all / waves), whatever rows they belong to, so
// that long and short rows fill the card alike; where a wave's run crosses
// from one (row, kv head) to the next it leaves one triple for each.
struct Cut {
    int prefix_tiles, chunk_tiles, chunks, blocks, waves;
    float2 *prefix_stats, *own_stats;
    float *prefix_o, *own_o;
};

__device__ __forceinline__ uint32_t own_tokens(const PagedAttnArgs& a, uint32_t r) {
    const int n = a.lengths[r];
    return n < 0 ? 0 : min((uint32_t)n, a.stride * a.pool.page_tokens.d);
}
template <int TILE>
__device__ __forceinline__ uint32_t own_tiles(const PagedAttnArgs& a, uint32_t r) {
    return (own_tokens(a, r) + TILE - 1) / TILE;
}

template <bool IO, bool KV, int D, int MT>
__device__ __forceinline__ void prefix_block(const PagedAttnArgs& a, const Cut& c, int id, char* lds) {
    using F = Form<IO, KV, D>;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, quarter = lane >> 4, col = lane & 15;
    const int block = id % c.blocks, kvh = id / c.blocks % a.pool.kv_heads, chunk = id / c.blocks / a.pool.kv_heads;
    const int queries = (int)a.rows * a.group;
    struct {
        const void* base;
        const PagedAttnArgs& a;
        int first, last, kvh;
        __device__ size_t operator()(int m) const {
            const int f = min(first + m, last), r = f / a.group;
            return r * a.q_stride + (size_t)(kvh * a.group + f - r * a.group) * D;
        }
    } who{a.q, a, block * 16 * MT, queries - 1, kvh};
    stage_queries<IO, KV, D>((v4u*)lds, 16 * MT, tid, 256, who);
    __syncthreads();
    Sums<D, MT> s;
    s.clear();
    int bad = 0;
    const int first = chunk * c.chunk_tiles;
    add_tiles<IO, KV, D, MT>(a, (const v4u*)lds, 16 * MT, a.prefix, a.prefix_tokens, first + wave,
                             min(first + c.chunk_tiles, c.prefix_tiles), 4, kvh, s, bad);
    if (bad && a.status) atomicOr(a.status, bad);
    __syncthreads();
    // the four waves' sums: the common reference, then o in pairs
    float2* stats = (float2*)lds;  // [4][16 MT]
    v4f* part = (v4f*)(lds + 4 * 16 * MT * sizeof(float2));
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        s.l[m] += __shfl_xor(s.l[m], 16, kWave);
        s.l[m] += __shfl_xor(s.l[m], 32, kWave);
        if (quarter == 0) stats[wave * 16 * MT + 16 * m + col] = make_float2(s.ref[m], s.l[m]);
    }
    __syncthreads();
    float ref[MT], l[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        float2 x[4];
        ref[m] = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            x[w] = stats[w * 16 * MT + 16 * m + col];
            ref[m] = fmaxf(ref[m], x[w].x);
        }
        const float sub = ref[m] == -INFINITY ? 0.0f : ref[m];
        l[m] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) l[m] += x[w].y * __builtin_amdgcn_exp2f(x[w].x == ref[m] ? 0.0f : x[w].x - sub);
        const float mine = __builtin_amdgcn_exp2f(s.ref[m] == ref[m] ? 0.0f : s.ref[m] - sub);
#pragma unroll
        for (int f = 0; f < F::kFrags; ++f) s.o[m][f] *= mine;
    }
    auto put = [&](int to) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int f = 0; f < F::kFrags; ++f) part[((to * MT + m) * F::kFrags + f) * 64 + lane] = s.o[m][f];
    };
    auto add = [&](int from) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int f = 0; f < F::kFrags; ++f) s.o[m][f] += part[((from * MT + m) * F::kFrags + f) * 64 + lane];
    };
    if (wave >= 2) put(wave - 2);
    __syncthreads();
    if (wave < 2) add(wave);
    __syncthreads();
    if (wave == 1) put(0);
    __syncthreads();
    if (wave) return;
    add(0);
    const size_t at = ((size_t)(kvh * c.chunks + chunk) * c.blocks + block) * 16 * MT;
#pragma unroll
    for (int m = 0; m < MT; ++m)
        if (block * 16 * MT + 16 * m + col < queries)
            store_sums<F::kWide, D>(c.prefix_stats, c.prefix_o, at + 16 * m + col, s.o[m], ref[m], l[m], quarter);
}

template <bool IO, bool KV, int D>
__device__ __forceinline__ void own_block(const PagedAttnArgs& a, const Cut& c, int id, char* lds) {
    using F = Form<IO, KV, D>;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, quarter = lane >> 4, col = lane & 15;
    const int groups = c.waves / 4;
    // tiles before each row, in LDS: thread t sums rows [t * per, (t + 1) * per)
    uint32_t* ahead = (uint32_t*)lds;
    uint32_t* sums = ahead + a.rows + 1;
    const uint32_t per = (a.rows + 255) / 256;
    uint32_t mine = 0;
    int bad = 0;
    for (uint32_t r = tid * per; r < min((tid + 1) * per, a.rows); ++r) {
        mine += own_tiles<F::kTile>(a, r);
        if ((int)a.lengths[r] > 0 && (uint32_t)a.lengths[r] > a.stride * a.pool.page_tokens.d) bad |= ZG_STATUS_POSITION;
    }
    if (bad && a.status && id == 0) atomicOr(a.status, bad);
    uint32_t upto = mine;  // inclusive sum over the wave, then over the waves
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t x = (uint32_t)__shfl_up((int)upto, off, kWave);
        if (lane >= off) upto += x;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    uint32_t at = upto - mine;
    for (int w = 0; w < wave; ++w) at += sums[w];
    for (uint32_t r = tid * per; r < min((tid + 1) * per, a.rows); ++r) {
        ahead[r] = at;
        at += own_tiles<F::kTile>(a, r);
    }
    const uint32_t all = sums[0] + sums[1] + sums[2] + sums[3];
    if (tid == 0) ahead[a.rows] = all;
    __syncthreads();
    const uint32_t kvs = a.pool.kv_heads, total = all * kvs;
    const uint32_t run = (total + c.waves - 1) / c.waves;
    // neighbouring runs lie on different CUs
    const uint32_t w = wave * groups + id;
    uint32_t t = w * run;
    const uint32_t end = min(t + run, total);
    if (t >= end) return;
    // the row that holds tile t: the last one with ahead[row] * kvs <= t
    uint32_t r = 0;
    for (uint32_t lo = 0, hi = a.rows; hi - lo > 1;) {
        const uint32_t mid = (lo + hi) / 2;
        if (ahead[mid] * kvs <= t) lo = r = mid;
        else hi = mid;
    }
    v4u* queries = (v4u*)(lds + (((a.rows + 5) * 4 + 15) & ~15u)) + wave * F::kParts * F::kSteps * 4 * a.group;
    bad = 0;
    while (t < end) {
        const uint32_t n = ahead[r + 1] - ahead[r];
        if (ahead[r + 1] * kvs <= t) {
            ++r;
            continue;
        }
        const uint32_t in_row = t - ahead[r] * kvs, kvh = in_row / n, tile = in_row - kvh * n;
        const uint32_t upto_tile = min(n, tile + (end - t));
        struct {
            const void* base;
            size_t first;
            __device__ size_t operator()(int m) const { return first + (size_t)m * D; }
        } who{a.q, r * a.q_stride + (size_t)kvh * a.group * D};
        stage_queries<IO, KV, D>(queries, a.group, lane, 64, who);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        Sums<D, 1> s;
        s.clear();
        add_tiles<IO, KV, D, 1>(a, queries, a.group, a.table + (size_t)r * a.stride, own_tokens(a, r), (int)tile,
                                (int)upto_tile, 1, (int)kvh, s, bad);
        __builtin_amdgcn_wave_barrier();
        s.l[0] += __shfl_xor(s.l[0], 16, kWave);
        s.l[0] += __shfl_xor(s.l[0], 32, kWave);
        if (col < a.group)
            store_sums<F::kWide, D>(c.own_stats, c.own_o, ((size_t)w + r * kvs + kvh) * a.group + col, s.o[0], s.ref[0],
                                    s.l[0], quarter);
        t += upto_tile - tile;
    }
    if (bad && a.status) atomicOr(a.status, bad);
}

template <bool IO, bool KV, int D, int MT>
__global__ __launch_bounds__(256, MT * D > 128 ? 1 : 2) void paged_attn_kernel(PagedAttnArgs a, Cut c) {
    extern __shared__ __align__(16) char lds[];
    const int over_prefix = c.chunks * c.blocks * a.pool.kv_heads;
    if ((int)blockIdx.x < over_prefix) prefix_block<IO, KV, D, MT>(a, c, blockIdx.x, lds);
    else own_block<IO, KV, D>(a, c, blockIdx.x - over_prefix, lds);
}

// Workgroup (query head, row, 64 elements): lane group tid / 16 joins the
// pieces tid / 16, + 16, ... in their order, the prefix's first.
template <bool IO, int D, int TILE>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a, Cut c, int mt) {
    extern __shared__ float weight[];  // per piece
    __shared__ uint32_t sums[2][4];
    __shared__ float tops[4], ls[4];
    __shared__ v4f parts[16][16];
    const uint32_t h = blockIdx.x, r = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (a.lengths[r] < 0) return;
    const uint32_t kvs = a.pool.kv_heads, kvh = h / a.group, in_group = h - kvh * a.group;
    uint32_t before = 0, all = 0;
    for (uint32_t i = tid; i < a.rows; i += 256) {
        const uint32_t n = own_tiles<TILE>(a, i);
        all += n;
        if (i < r) before += n;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        before += (uint32_t)__shfl_xor((int)before, off, kWave);
        all += (uint32_t)__shfl_xor((int)all, off, kWave);
    }
    if (lane == 0) {
        sums[0][wave] = before;
        sums[1][wave] = all;
    }
    __syncthreads();
    before = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3];
    all = sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
    const uint32_t run = (all * kvs + c.waves - 1) / c.waves, n = own_tiles<TILE>(a, r);
    const uint32_t tile = before * kvs + kvh * n;
    const uint32_t first = n ? tile / run : 0, own = n ? (tile + n - 1) / run - first + 1 : 0;
    const uint32_t pieces = c.chunks + own;
    const uint32_t f = r * a.group + in_group;
    auto prefix_at = [&](uint32_t i) { return ((size_t)(kvh * c.chunks + i) * c.blocks) * 16 * mt + f; };
    auto own_at = [&](uint32_t i) { return ((size_t)first + i + r * kvs + kvh) * a.group + in_group; };
    float top = -INFINITY;
    for (uint32_t i = tid; i < pieces; i += 256)
        top = fmaxf(top, i < (uint32_t)c.chunks ? c.prefix_stats[prefix_at(i)].x : c.own_stats[own_at(i - c.chunks)].x);
    top = wave_max(top);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float sub = top == -INFINITY ? 0.0f : top;
    float l = 0.0f;
    for (uint32_t i = tid; i < pieces; i += 256) {
        const float2 x = i < (uint32_t)c.chunks ? c.prefix_stats[prefix_at(i)] : c.own_stats[own_at(i - c.chunks)];
        const float e = __builtin_amdgcn_exp2f(x.x == top ? 0.0f : x.x - sub);
        weight[i] = e;
        l += e * x.y;
    }
    l = wave_sum_xor(l, kWave);
    if (lane == 0) ls[wave] = l;
    __syncthreads();
    l = (ls[0] + ls[1]) + (ls[2] + ls[3]);
    const int e = blockIdx.z * 64 + 4 * (tid & 15);
    v4f o = {};
    for (uint32_t i = tid >> 4; i < pieces; i += 16) {
        const float* from = i < (uint32_t)c.chunks ? c.prefix_o + prefix_at(i) * D : c.own_o + own_at(i - c.chunks) * D;
        o += weight[i] * *(const v4f*)(from + e);
    }
    parts[tid >> 4][tid & 15] = o;
    __syncthreads();
    if (tid >= 16) return;
    o = parts[0][tid];
#pragma unroll
    for (int i = 1; i < 16; ++i) o += parts[i][tid];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = l == 0.0f ? 0.0f : o[j] / l;
    store4<IO>(a.out, r * a.out_stride + (size_t)h * D + e, o);
}

// ------------------------------------------------------------------- host

// Tiles of 16 queries that share a pass over the prefix: their sums take
// MT * D / 4 registers a lane of the 512.
static int tiles_of_queries(uint32_t rows, int group, int head_dim) {
    const uint64_t n = (uint64_t)rows * group;
    return n <= 16 ? 1 : n <= 32 || head_dim == 256 ? 2 : 4;
}

static Cut cut_of(uint32_t rows, int q_heads, int kv_heads, int head_dim, int tile, uint32_t prefix_tokens,
                  uint64_t row_tokens, void* workspace, size_t* bytes) {
    Cut c{};
    const int group = q_heads / kv_heads, mt = tiles_of_queries(rows, group, head_dim);
    c.blocks = (int)(((uint64_t)rows * group + 16 * mt - 1) / (16 * mt));
    c.prefix_tiles = (int)((prefix_tokens + tile - 1) / tile);
    if (c.prefix_tiles) {
        const int most = (c.prefix_tiles + 3) / 4;  // four tiles: one a wave
        const int want = std::max(1, std::min(most, kPrefixGroups / std::max(1, kv_heads * c.blocks)));
        c.chunk_tiles = (c.prefix_tiles + want - 1) / want;
        c.chunks = (c.prefix_tiles + c.chunk_tiles - 1) / c.chunk_tiles;
    }
    const uint64_t own_tiles = (uint64_t)rows * kv_heads * ((row_tokens + tile - 1) / tile);
    c.waves = 4 * (int)std::min<uint64_t>(kOwnGroups, own_tiles);
    const size_t prefix_rows = (size_t)kv_heads * c.chunks * c.blocks * 16 * mt;
    const size_t own_rows = ((size_t)c.waves + (size_t)rows * kv_heads) * group;
    char* at = (char*)workspace;
    auto take = [&](size_t n) {
        char* p = at;
        at += (n + 255) / 256 * 256;
        return p;
    };
    c.prefix_stats = (float2*)take(prefix_rows * sizeof(float2));
    c.own_stats = (float2*)take(own_rows * sizeof(float2));
    c.prefix_o = (float*)take(prefix_rows * head_dim * sizeof(float));
    c.own_o = (float*)take(own_rows * head_dim * sizeof(float));
    if (bytes) *bytes = (size_t)(at - (char*)workspace);
    return c;
}

size_t paged_attn_workspace(uint32_t rows, int q_heads, int kv_heads, int head_dim, int bf16, uint32_t prefix_tokens,
                            uint64_t row_tokens) {
    size_t bytes = 0;
    cut_of(rows, q_heads, kv_heads, head_dim, bf16 ? 32 : 16, prefix_tokens, row_tokens, nullptr, &bytes);
    return bytes;
}

template <bool IO, bool KV, int D, int MT>
static hipError_t launch(const PagedAttnArgs& a, const Cut& c, hipStream_t st) {
    using F = Form<IO, KV, D>;
    const size_t queries = (size_t)F::kParts * F::kSteps * 4 * 16;  // bytes of a query, 16 a step and part and quarter
    const size_t prefix = c.chunks ? std::max(queries * 16 * MT, (size_t)4 * 16 * MT * 8 + (size_t)2 * MT * D * 64) : 0;
    const size_t own = ((a.rows + 5) * 4 + 15) / 16 * 16 + 4 * a.group * queries;
    const size_t lds = std::max(prefix, own);
    auto kernel = paged_attn_kernel<IO, KV, D, MT>;
    if (lds > 65536) {
        hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    kernel<<<c.chunks * c.blocks * a.pool.kv_heads + c.waves / 4, 256, lds, st>>>(a, c);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    paged_join_kernel<IO, D, F::kTile><<<dim3(a.q_heads, a.rows, D / 64), 256, (c.chunks + c.waves) * sizeof(float), st>>>(a, c, MT);
    return hipGetLastError();
}

hipError_t paged_attn(const PagedAttnArgs& a, hipStream_t st) {
    const Cut c = cut_of(a.rows, a.q_heads, a.pool.kv_heads, a.pool.head_dim, a.pool.bf16 ? 32 : 16, a.prefix_tokens,
                         (uint64_t)a.stride * a.pool.page_tokens.d, a.workspace, nullptr);
    const int mt = c.chunks ? tiles_of_queries(a.rows, a.group, a.pool.head_dim) : 1;
    auto by_tiles = [&](auto io, auto kv, auto dim) {
        constexpr bool IO = decltype(io)::value, KV = decltype(kv)::value;
        constexpr int D = decltype(dim)::value;
        if (mt == 1) return launch<IO, KV, D, 1>(a, c, st);
        if constexpr (D < 256)
            if (mt == 4) return launch<IO, KV, D, 4>(a, c, st);
        return launch<IO, KV, D, 2>(a, c, st);
    };
    auto by_dim = [&](auto io, auto kv) {
        switch (a.pool.head_dim) {
        case 64: return by_tiles(io, kv, std::integral_constant<int, 64>{});
        case 128: return by_tiles(io, kv, std::integral_constant<int, 128>{});
        default: return by_tiles(io, kv, std::integral_constant<int, 256>{});
        }
    };
    if (a.io_bf16) return a.pool.bf16 ? by_dim(std::true_type{}, std::true_type{}) : by_dim(std::true_type{}, std::false_type{});
    return a.pool.bf16 ? by_dim(std::false_type{}, std::true_type{}) : by_dim(std::false_type{}, std::false_type{});
}

}  // namespace zg

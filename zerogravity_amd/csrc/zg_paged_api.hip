// Entry points of the paged KV cache and of the logits readout
// (include/zg_hip.h): argument checks, then the kernels of zg_paged.hip,
// zg_paged_attn.hip and zg_logits.hip.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <exception>
#include <string>

#include "zg_context.hpp"
#include "zg_paged.hpp"

using zgc::fail;

namespace {

constexpr size_t kMaxRows = 4096;
constexpr size_t kMaxRowTokens = (size_t)1 << 30;
constexpr size_t kMaxTokens = ((size_t)1 << 24) - 1;  // of 256 threads each in one launch
constexpr size_t kMaxHistory = (size_t)1 << 28;  // what zg_logits.hip's words count
constexpr size_t kMaxStride = (size_t)1 << 32;  // elements: offsets of 2^31 rows stay within 64 bits

// The context's device for the length of a call; the caller's comes back.
struct OnDevice {
    int before = -1;
    bool ok = true;
    explicit OnDevice(int device) {
        if (hipGetDevice(&before) != hipSuccess) before = -1;
        if (before == device) before = -1;  // nothing to bring back
        else ok = hipSetDevice(device) == hipSuccess;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

// A refusal: a status code and its reason.
struct Refusal {
    int code = ZG_COMPLETED;
    const char* why = "";
    explicit operator bool() const { return code != ZG_COMPLETED; }
};

bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

Refusal check_pool(const zg_paged_kv* c) {
    if (!c || !c->keys || !c->values || !aligned(c->keys, 16) || !aligned(c->values, 16))
        return {ZG_E_MALFORMED, "paged cache pointers"};
    if (c->pages == 0 || c->page_tokens == 0 || c->kv_heads == 0)
        return {ZG_E_MALFORMED, "paged cache without pages, slots or heads"};
    if (c->dtype != ZG_BF16 && c->dtype != ZG_F32) return {ZG_E_UNSUPPORTED, "paged cache of ZG_BF16 or ZG_F32"};
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return {ZG_E_UNSUPPORTED, "paged cache offered for head_dim 64, 128 and 256"};
    if (c->page_tokens > 65536 || c->kv_heads > 1024 || c->pages > 0x7fffffffu)
        return {ZG_E_LIMIT, "paged cache of at most 65536 tokens a page, 1024 heads and 2^31 - 1 pages"};
    if (c->page_stride % 64 || c->page_stride < c->page_tokens * c->kv_heads * c->head_dim)
        return {ZG_E_MALFORMED, "page stride is a multiple of 64 that holds a page"};
    // slot offsets are counted in 64 elements and held in 32 bits
    if (c->page_stride / 64 > 0xffffffffu / c->pages) return {ZG_E_LIMIT, "paged cache of at most 2^38 elements"};
    return {};
}

Refusal check_rows(const zg_paged_kv* c, const zg_paged_rows* r) {
    if (!r || !r->pages || r->rows == 0 || r->stride == 0) return {ZG_E_MALFORMED, "page tables"};
    if (r->rows > kMaxRows) return {ZG_E_LIMIT, "at most 4096 rows"};
    if (r->stride > kMaxRowTokens / c->page_tokens || r->prefix_tokens > kMaxRowTokens)
        return {ZG_E_LIMIT, "page tables of at most 2^30 tokens a row"};
    return {};
}

Refusal check_attention(const zg_paged_kv* c, const zg_paged_rows* r, size_t q_heads) {
    if (Refusal why = check_pool(c)) return why;
    if (Refusal why = check_rows(c, r)) return why;
    if (r->prefix_tokens && !r->prefix) return {ZG_E_MALFORMED, "a prefix without its pages"};
    if (q_heads == 0 || q_heads % c->kv_heads) return {ZG_E_MALFORMED, "query heads are a multiple of the kv heads"};
    // the rows' tiles of 16 or 32 tokens are counted in 32 bits
    if ((r->stride * c->page_tokens + 15) / 16 >= ((size_t)1 << 31) / (r->rows * c->kv_heads))
        return {ZG_E_LIMIT, "rows * kv_heads * tokens a row can hold is at most 2^35"};
    if (q_heads / c->kv_heads > 16) return {ZG_E_UNSUPPORTED, "at most 16 query heads to a kv head"};
    return {};
}

zg::PagedPool pool_of(const zg_paged_kv* c) {
    zg::PagedPool p;
    p.keys = c->keys;
    p.values = c->values;
    p.pages = (uint32_t)c->pages;
    p.page_tokens = zg::FastDiv::of((uint32_t)c->page_tokens);
    p.page_units = (uint32_t)(c->page_stride / 64);
    p.slot_units = (uint32_t)(c->kv_heads * c->head_dim / 64);
    p.kv_heads = (int)c->kv_heads;
    p.head_dim = (int)c->head_dim;
    p.bf16 = c->dtype == ZG_BF16;
    return p;
}

// One call on a context: its lock, its device, and no exception past the C
// boundary.
template <typename F>
int on_context(zg_ctx* ctx, F body) {
    if (!ctx) return ZG_E_MALFORMED;
    try {
        std::lock_guard<std::recursive_mutex> g(ctx->mu);
        OnDevice device(ctx->device);
        if (!device.ok) return fail(ctx, ZG_E_DEVICE, "the context's device is not available");
        return body();
    } catch (...) {
        return ZG_E_RESOURCE;
    }
}

int refuse(zg_ctx* ctx, const Refusal& r) { return fail(ctx, r.code, r.why); }

}  // namespace

extern "C" {

int zg_paged_admit(const zg_paged_kv* cache, const zg_paged_rows* rows, const int32_t* lengths, size_t q_heads,
                   char* msg, size_t msg_len) {
    char text[160] = "";
    auto check = [&]() -> int {
        if (Refusal why = check_attention(cache, rows, q_heads)) {
            snprintf(text, sizeof text, "%s", why.why);
            return why.code;
        }
        if (!lengths) {
            snprintf(text, sizeof text, "lengths");
            return ZG_E_MALFORMED;
        }
        auto page_ok = [&](int32_t p) { return p >= 0 && (size_t)p < cache->pages; };
        const size_t pt = cache->page_tokens;
        for (size_t i = 0; i < (rows->prefix_tokens + pt - 1) / pt; ++i)
            if (!page_ok(rows->prefix[i])) {
                snprintf(text, sizeof text, "prefix page %zu is %d, outside the pool", i, (int)rows->prefix[i]);
                return ZG_E_MALFORMED;
            }
        for (size_t r = 0; r < rows->rows; ++r) {
            if (lengths[r] <= 0) continue;
            const size_t n = (size_t)lengths[r], used = (n + pt - 1) / pt;
            if (used > rows->stride) {
                snprintf(text, sizeof text, "row %zu holds %zu tokens, past its %zu pages", r, n, rows->stride);
                return ZG_E_MALFORMED;
            }
            for (size_t i = 0; i < used; ++i)
                if (!page_ok(rows->pages[r * rows->stride + i])) {
                    snprintf(text, sizeof text, "row %zu: page %zu is %d, outside the pool", r, i,
                             (int)rows->pages[r * rows->stride + i]);
                    return ZG_E_MALFORMED;
                }
        }
        return ZG_COMPLETED;
    };
    const int rc = check();
    if (msg && msg_len) snprintf(msg, msg_len, "%s", text);
    return rc;
}

int zg_paged_append_device(zg_ctx* ctx, const zg_paged_kv* cache, const zg_paged_rows* rows, size_t tokens,
                           size_t q_heads, const void* q, size_t q_stride, size_t q_head_stride, const void* k,
                           size_t k_stride, const void* v, size_t v_stride, int dtype, const float* q_norm,
                           const float* k_norm, float eps, size_t rotate, float theta_scale, const int32_t* positions,
                           const int32_t* token_rows, void* q_out, int32_t* status, void* stream) {
    return on_context(ctx, [&]() -> int {
        if (Refusal why = check_pool(cache)) return refuse(ctx, why);
        if (Refusal why = check_rows(cache, rows)) return refuse(ctx, why);
        if (dtype != ZG_F32 && dtype != ZG_BF16)
            return fail(ctx, ZG_E_UNSUPPORTED, "paged append of ZG_F32 or ZG_BF16 activations");
        const size_t four = dtype == ZG_BF16 ? 8 : 16, width = cache->kv_heads * cache->head_dim;
        if (!k || !v || !positions || tokens == 0 || k_stride < width || v_stride < width || k_stride % 4 ||
            v_stride % 4 || !aligned(k, four) || !aligned(v, four))
            return fail(ctx, ZG_E_MALFORMED, "paged append: keys, values and positions");
        if (q_heads > 65536 || tokens > kMaxTokens || std::max({q_stride, q_head_stride, k_stride, v_stride}) > kMaxStride)
            return fail(ctx, ZG_E_LIMIT, "paged append of at most 2^24 - 1 tokens, 65536 query heads and strides of 2^32");
        if ((q_heads == 0) != (q == nullptr) || (q_heads == 0) != (q_out == nullptr) || q_head_stride % 4 ||
            q_stride % 4 || !aligned(q, four) || !aligned(q_out, four) ||
            (q_heads && (q_head_stride < cache->head_dim || q_stride < (q_heads - 1) * q_head_stride + cache->head_dim)))
            return fail(ctx, ZG_E_MALFORMED, "paged append: queries");
        if (rotate > cache->head_dim || rotate % 8 || !(theta_scale > 0.0f && theta_scale <= 1.0f))
            return fail(ctx, ZG_E_MALFORMED, "paged append: the rotation takes a multiple of 8 elements of a head");
        if ((q_norm || k_norm) && !(eps > 0.0f && std::isfinite(eps)))
            return fail(ctx, ZG_E_MALFORMED, "paged append: a norm's eps is positive");
        if (!aligned(q_norm, 16) || !aligned(k_norm, 16)) return fail(ctx, ZG_E_MALFORMED, "paged append: norm alignment");
        if (!token_rows && tokens > rows->rows)
            return fail(ctx, ZG_E_MALFORMED, "paged append: more tokens than rows need token_rows");
        if (q && q == q_out && (q_head_stride != cache->head_dim || q_stride != q_heads * cache->head_dim))
            return fail(ctx, ZG_E_MALFORMED, "paged append: queries in place are contiguous");
        zg::AppendArgs a;
        a.pool = pool_of(cache);
        a.table = rows->pages;
        a.rows = (uint32_t)rows->rows;
        a.stride = (uint32_t)rows->stride;
        a.prefix_tokens = (uint32_t)rows->prefix_tokens;
        a.tokens = tokens;
        a.q_heads = (int)q_heads;
        a.q = q;
        a.k = k;
        a.v = v;
        a.q_stride = q_stride;
        a.q_head_stride = q_head_stride;
        a.k_stride = k_stride;
        a.v_stride = v_stride;
        a.io_bf16 = dtype == ZG_BF16;
        a.q_norm = q_norm;
        a.k_norm = k_norm;
        a.eps = eps;
        a.rotate = (int)rotate;
        a.theta_scale = theta_scale;
        a.positions = positions;
        a.token_rows = token_rows;
        a.q_out = q_out;
        a.status = status;
        ZG_HIP(zg::paged_append(a, stream ? (hipStream_t)stream : ctx->stream));
        return ZG_COMPLETED;
    });
}

size_t zg_paged_attn_workspace_bytes(const zg_paged_kv* cache, const zg_paged_rows* rows, size_t q_heads) {
    if (check_attention(cache, rows, q_heads)) return 0;
    return zg::paged_attn_workspace((uint32_t)rows->rows, (int)q_heads, (int)cache->kv_heads, (int)cache->head_dim, cache->dtype == ZG_BF16,
                                    (uint32_t)rows->prefix_tokens, (uint64_t)rows->stride * cache->page_tokens);
}

int zg_paged_attn_device(zg_ctx* ctx, const zg_paged_kv* cache, const zg_paged_rows* rows, const int32_t* lengths,
                         size_t q_heads, const void* q, size_t q_stride, int dtype, float scale, void* workspace,
                         void* out, size_t out_stride, int32_t* status, void* stream) {
    return on_context(ctx, [&]() -> int {
        if (Refusal why = check_attention(cache, rows, q_heads)) return refuse(ctx, why);
        if (dtype != ZG_F32 && dtype != ZG_BF16)
            return fail(ctx, ZG_E_UNSUPPORTED, "paged attention of ZG_F32 or ZG_BF16 queries");
        const size_t width = q_heads * cache->head_dim;
        if (!lengths || !q || !out || !workspace || q_stride < width || out_stride < width || q_stride % 8 ||
            out_stride % 8 || !aligned(q, 16) || !aligned(out, 16) || !aligned(workspace, 16))
            return fail(ctx, ZG_E_MALFORMED, "paged attention: queries, lengths, workspace and outputs");
        if (std::max(q_stride, out_stride) > kMaxStride)
            return fail(ctx, ZG_E_LIMIT, "paged attention with strides of at most 2^32");
        if (!std::isfinite(2.0f * scale))  // the kernels count in log2
            return fail(ctx, ZG_E_MALFORMED, "paged attention: twice the scale is finite");
        if (q == out && q_stride != out_stride)
            return fail(ctx, ZG_E_MALFORMED, "paged attention: outputs in place keep the queries' stride");
        zg::PagedAttnArgs a;
        a.pool = pool_of(cache);
        a.table = rows->pages;
        a.lengths = lengths;
        a.prefix = rows->prefix;
        a.rows = (uint32_t)rows->rows;
        a.stride = (uint32_t)rows->stride;
        a.prefix_tokens = (uint32_t)rows->prefix_tokens;
        a.q_heads = (int)q_heads;
        a.group = (int)(q_heads / cache->kv_heads);
        a.q = q;
        a.q_stride = q_stride;
        a.io_bf16 = dtype == ZG_BF16;
        a.scale = scale;
        a.workspace = workspace;
        a.out = out;
        a.out_stride = out_stride;
        a.status = status;
        ZG_HIP(zg::paged_attn(a, stream ? (hipStream_t)stream : ctx->stream));
        return ZG_COMPLETED;
    });
}

size_t zg_logits_adjust_workspace_bytes(size_t rows, size_t vocab) {
    if (rows == 0 || rows > 65535 || vocab == 0 || vocab > ((size_t)1 << 30)) return 0;
    return zg::logits_workspace(rows, vocab);
}

int zg_logits_adjust_device(zg_ctx* ctx, size_t rows, size_t vocab, const void* logits, size_t ld, int dtype,
                            const zg_logit_rules* rules, void* out, size_t out_ld, uint32_t* greedy, int record,
                            void* workspace, int32_t* status, void* stream) {
    return on_context(ctx, [&]() -> int {
        if (dtype != ZG_F32 && dtype != ZG_BF16)
            return fail(ctx, ZG_E_UNSUPPORTED, "logits of ZG_F32 or ZG_BF16");
        const size_t size = dtype == ZG_BF16 ? 2 : 4;
        if (!logits || !out || !rules || rows == 0 || vocab == 0 || ld < vocab || out_ld < vocab ||
            !aligned(logits, size) || !aligned(out, size) || (logits == out && ld != out_ld))
            return fail(ctx, ZG_E_MALFORMED, "logits, their strides and rules");
        if (rows > 65535 || vocab > ((size_t)1 << 30))
            return fail(ctx, ZG_E_LIMIT, "logits of at most 65535 rows and a vocabulary of 2^30");
        const zg_logit_rules& u = *rules;
        if (std::max({ld, out_ld, u.mask_stride, u.mask_rows}) > kMaxStride)
            return fail(ctx, ZG_E_LIMIT, "logits and masks with strides of at most 2^32");
        if ((u.history == nullptr) != (u.history_lengths == nullptr) ||
            (u.history && (u.history_stride == 0 || u.history_stride > kMaxHistory)) ||
            (!u.history && (u.prompt_lengths || u.repetition || u.frequency || u.presence)))
            return fail(ctx, ZG_E_MALFORMED, "penalties need a history of 1 to 2^28 tokens a row and its lengths");
        if ((u.bias_ids == nullptr) != (u.bias_values == nullptr) || (u.bias_ids == nullptr) != (u.bias_lengths == nullptr) ||
            (u.bias_ids && u.bias_stride == 0))
            return fail(ctx, ZG_E_MALFORMED, "biases need ids, values and lengths");
        if (u.bias_ids && u.bias_stride > 65535) return fail(ctx, ZG_E_LIMIT, "at most 65535 biases a row");
        if (u.masks ? u.mask_rows == 0 || u.mask_stride < (vocab + 31) / 32 || (!u.mask_of && u.mask_rows < rows)
                    : u.mask_of != nullptr)
            return fail(ctx, ZG_E_MALFORMED, "masks hold a bit for every token, one row for each mask");
        if ((record != 0 && record != 1) || (record && (!u.history || !greedy)))
            return fail(ctx, ZG_E_MALFORMED, "recording needs a history and greedy ids");
        if (greedy && (!workspace || !aligned(workspace, 16)))
            return fail(ctx, ZG_E_MALFORMED, "greedy ids need a workspace");
        zg::LogitArgs a;
        a.rows = rows;
        a.vocab = vocab;
        a.logits = logits;
        a.ld = ld;
        a.bf16 = dtype == ZG_BF16;
        a.rules = u;
        a.out = out;
        a.out_ld = out_ld;
        a.greedy = greedy;
        a.record = record;
        a.workspace = workspace;
        a.status = status;
        ZG_HIP(zg::logits_adjust(a, stream ? (hipStream_t)stream : ctx->stream));
        return ZG_COMPLETED;
    });
}

}  // extern "C"

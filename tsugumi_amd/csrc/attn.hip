// attn.hip — the attention half of a decoder layer over a paged key/value
// cache: the plan object, the checks, and the append (head norms, rotation,
// cache write).
#include "attn_internal.hpp"

#include <cmath>
#include <new>

namespace tsg {
namespace {

constexpr uint32_t kMaxHeads = 1024;
constexpr uint32_t kMaxHeadDim = 512;
constexpr uint32_t kMinPage = 16, kMaxPage = 4096;
constexpr uint64_t kMaxCapacity = 1u << 30;  // tokens a page table may hold
constexpr uint32_t kMaxAttnRows = 1u << 22;

bool is16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool is4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
bool is2(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1u) == 0; }

uint32_t cell_bytes(const tsg_attn_config& c) { return c.kv_type == TSG_KV_E4M3 ? 1u : 2u; }

}  // namespace

tsg_status check_attn_config(const tsg_attn_config* c) {
    TSG_REQUIRE(c, TSG_ERR_INVALID_ARGUMENT, "attention config is NULL");
    TSG_REQUIRE(c->kv_heads > 0 && c->q_heads > 0 && c->q_heads <= kMaxHeads,
                TSG_ERR_INVALID_ARGUMENT, "head counts must be in 1...%u", kMaxHeads);
    TSG_REQUIRE(c->q_heads % c->kv_heads == 0, TSG_ERR_INVALID_ARGUMENT,
                "%u query heads do not share %u key heads evenly", c->q_heads, c->kv_heads);
    TSG_REQUIRE(c->kv_type == TSG_KV_F16 || c->kv_type == TSG_KV_E4M3, TSG_ERR_INVALID_ARGUMENT,
                "unknown cache type %d", (int)c->kv_type);
    const uint32_t step = 16u / cell_bytes(*c);
    TSG_REQUIRE(c->head_dim > 0 && c->head_dim <= kMaxHeadDim && c->head_dim % step == 0,
                TSG_ERR_UNSUPPORTED, "head_dim %u: a multiple of %u up to %u (16-byte cache rows)",
                c->head_dim, step, kMaxHeadDim);
    TSG_REQUIRE(c->page_tokens >= kMinPage && c->page_tokens <= kMaxPage &&
                    (c->page_tokens & (c->page_tokens - 1u)) == 0,
                TSG_ERR_UNSUPPORTED, "page_tokens %u: a power of two in %u...%u", c->page_tokens,
                kMinPage, kMaxPage);
    TSG_REQUIRE(c->window <= kMaxCapacity && c->sinks <= kMaxCapacity, TSG_ERR_INVALID_ARGUMENT,
                "window or sinks above %llu", (unsigned long long)kMaxCapacity);
    TSG_REQUIRE(c->window > 0 || c->sinks == 0, TSG_ERR_INVALID_ARGUMENT,
                "sinks without a window: every token is visible already");
    TSG_REQUIRE(std::isfinite(c->scale) && std::fabs(c->scale) <= 1e6f, TSG_ERR_INVALID_ARGUMENT,
                "scale must be finite and at most 1e6");
    // the scales' own reciprocals and products with `scale` stay normal fp32
    const auto scale_ok = [](float s) { return s >= 1e-6f && s <= 1e6f; };
    TSG_REQUIRE(scale_ok(c->k_scale) && scale_ok(c->v_scale), TSG_ERR_INVALID_ARGUMENT,
                "k_scale and v_scale must be in 1e-6...1e6");
    TSG_REQUIRE(c->kv_type == TSG_KV_E4M3 || (c->k_scale == 1.0f && c->v_scale == 1.0f),
                TSG_ERR_INVALID_ARGUMENT, "an fp16 cache takes no scales (k_scale = v_scale = 1)");
    return TSG_OK;
}

tsg_status check_attn_pages(const tsg_attn_config& c, const tsg_kv_pages* p) {
    TSG_REQUIRE(p && p->k && p->v, TSG_ERR_INVALID_ARGUMENT, "NULL cache pages");
    TSG_REQUIRE(p->num_pages > 0, TSG_ERR_INVALID_ARGUMENT, "a cache needs at least one page");
    const uint32_t step = 16u / cell_bytes(c);
    TSG_REQUIRE(is16(p->k) && is16(p->v), TSG_ERR_ALIGNMENT, "cache pages must be 16-byte aligned");
    TSG_REQUIRE(p->token_stride % step == 0 && p->head_stride % step == 0 &&
                    p->page_stride % step == 0,
                TSG_ERR_ALIGNMENT, "cache strides must be multiples of 16 bytes");
    // 64-bit products: page_tokens <= 2^12, token_stride < 2^32, heads <= 2^10
    TSG_REQUIRE(p->head_stride < (1ull << 40) && p->page_stride < (1ull << 44),
                TSG_ERR_INVALID_ARGUMENT, "cache stride too large");
    const uint64_t run = (uint64_t)(c.page_tokens - 1u) * p->token_stride + c.head_dim;
    const uint64_t across = (uint64_t)(c.kv_heads - 1u) * p->head_stride;
    TSG_REQUIRE(p->token_stride >= c.head_dim, TSG_ERR_INVALID_ARGUMENT, "token stride is too small");
    TSG_REQUIRE(c.kv_heads == 1 || p->head_stride >= run ||
                    (p->head_stride >= c.head_dim && p->token_stride >= across + c.head_dim),
                TSG_ERR_INVALID_ARGUMENT, "head stride is too small: heads overlap");
    TSG_REQUIRE(p->num_pages == 1 || p->page_stride >= run + across, TSG_ERR_INVALID_ARGUMENT,
                "page stride is too small: pages overlap");
    // the kernels address a head's tokens within a page by 32-bit byte offsets
    TSG_REQUIRE(run * cell_bytes(c) <= 0x7fffffffu, TSG_ERR_UNSUPPORTED,
                "a page's rows of one head must span less than 2 GiB");
    return TSG_OK;
}

tsg_status check_attn_batch(const tsg_attn_config& c, const tsg_attn_batch* b) {
    TSG_REQUIRE(b, TSG_ERR_INVALID_ARGUMENT, "attention batch is NULL");
    TSG_REQUIRE(b->num_seqs > 0, TSG_ERR_INVALID_ARGUMENT, "numSeqs must be positive");
    TSG_REQUIRE(b->rows > 0 && b->rows <= kMaxAttnRows, TSG_ERR_INVALID_ARGUMENT,
                "rows must be in 1...%u", kMaxAttnRows);
    TSG_REQUIRE(b->num_seqs <= kMaxAttnRows, TSG_ERR_INVALID_ARGUMENT, "too many sequences");
    TSG_REQUIRE(b->page_table && b->lengths, TSG_ERR_INVALID_ARGUMENT,
                "NULL page table or lengths");
    TSG_REQUIRE(is4(b->page_table) && is4(b->lengths) && is4(b->row_starts), TSG_ERR_ALIGNMENT,
                "page table, lengths and row starts must be 4-byte aligned");
    TSG_REQUIRE(b->table_stride > 0 && (uint64_t)b->table_stride * c.page_tokens <= kMaxCapacity,
                TSG_ERR_INVALID_ARGUMENT, "a page table holds 1...%llu tokens",
                (unsigned long long)kMaxCapacity);
    TSG_REQUIRE(b->row_starts || b->rows % b->num_seqs == 0, TSG_ERR_INVALID_ARGUMENT,
                "%u rows do not divide over %u sequences (give row starts)", b->rows, b->num_seqs);
    return TSG_OK;
}

// Whether rows of `a` and of `b` share an element, where that is plain: rows of
// one stride, single rows, or one address.
static bool rows_share(const uint16_t* a, uint64_t a_stride, uint64_t a_width, const uint16_t* b,
                       uint64_t b_stride, uint64_t b_width, uint64_t rows) {
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a) / 2u, pb = reinterpret_cast<uintptr_t>(b) / 2u;
    if (pa == pb) return true;
    const bool a_first = pa < pb;
    const uint64_t apart = a_first ? pb - pa : pa - pb;
    const uint64_t width = a_first ? a_width : b_width, other = a_first ? b_width : a_width;
    if (rows == 1u) return apart < width;
    if (a_stride != b_stride || apart >= (rows - 1u) * a_stride + width) return false;
    const uint64_t off = apart % a_stride;  // of the other's row in the first's
    return off < width || off + other > a_stride;
}

tsg_status attn_args(const tsg_attn* attn, const tsg_kv_pages* pages, const tsg_attn_batch* batch,
                     const uint16_t* q, uint32_t q_stride, uint16_t* out, uint32_t out_stride,
                     AttnArgs* a) {
    TSG_REQUIRE(attn, TSG_ERR_INVALID_ARGUMENT, "attn is NULL");
    const tsg_attn_config& c = attn->cfg;
    if (tsg_status s = check_attn_pages(c, pages)) return s;
    if (tsg_status s = check_attn_batch(c, batch)) return s;
    TSG_REQUIRE(q && out, TSG_ERR_INVALID_ARGUMENT, "NULL attention operand");
    TSG_REQUIRE((uint64_t)batch->rows * attn->group <= 0x7fffffffu, TSG_ERR_UNSUPPORTED,
                "too many rows for groups of %u query heads", attn->group);
    TSG_REQUIRE(q_stride >= c.q_heads * c.head_dim, TSG_ERR_INVALID_ARGUMENT,
                "q stride is too small");
    TSG_REQUIRE(out_stride >= c.q_heads * c.head_dim, TSG_ERR_INVALID_ARGUMENT,
                "out stride is too small");
    TSG_REQUIRE(is16(q) && is16(out) && q_stride % 8u == 0 && out_stride % 8u == 0,
                TSG_ERR_ALIGNMENT, "q and out rows must be 16-byte aligned");
    const uint32_t width = c.q_heads * c.head_dim;
    TSG_REQUIRE((q == out && (q_stride == out_stride || batch->rows == 1u)) ||
                    !rows_share(q, q_stride, width, out, out_stride, width, batch->rows),
                TSG_ERR_INVALID_ARGUMENT, "out shares elements with q and is not q itself");
    a->q = q;
    a->out = out;
    a->k = static_cast<const uint8_t*>(pages->k);
    a->v = static_cast<const uint8_t*>(pages->v);
    a->table = batch->page_table;
    a->lengths = batch->lengths;
    a->row_starts = batch->row_starts;
    a->error = attn->ctx->counters + kSyncErrorWord;
    a->page_stride = pages->page_stride * attn->cell;
    a->head_stride = pages->head_stride * attn->cell;
    a->token_stride = pages->token_stride * attn->cell;
    a->q_stride = q_stride;
    a->out_stride = out_stride;
    a->table_stride = batch->table_stride;
    a->num_seqs = batch->num_seqs;
    a->rows = batch->rows;
    a->seq_rows = batch->row_starts ? 0u : batch->rows / batch->num_seqs;
    a->num_pages = pages->num_pages;
    a->q_heads = c.q_heads;
    a->kv_heads = c.kv_heads;
    a->group = attn->group;
    a->dim = c.head_dim;
    a->page_shift = attn->page_shift;
    a->window = c.window;
    a->sinks = c.sinks;
    const double scale = std::fabs((double)c.scale) * c.k_scale * 1.4426950408889634;
    a->scale_log2 = scale > 1e-30 ? (float)scale : 1e-30f;
    a->q_sign = c.scale < 0.0f ? 0x80008000u : 0u;
    a->v_scale = c.v_scale;
    return TSG_OK;
}

namespace {

// ------------------------------------------------------------------ append
//
// Head rows x of q and k: y = x w / sqrt(mean(x^2) + eps) in fp32, then the
// rotation of pairs (a, b) by t = position * inv_freq: (a cos t - b sin t,
// b cos t + a sin t), one rounding at the end (fp16, or e4m3 of y / scale). The
// angle is formed in fp64, in revolutions, and only its fraction goes to fp32
// (v_sin_f32 / v_cos_f32 take revolutions): at position 10^6 an fp32 product
// would be off by 0.03 rad, the fraction is off by 2^-25 of a turn. HBM bounds
// it: 11,207 rows of 32 + 8 + 8 heads of 128 (275 MB) 59 us, 4.6 TB/s; one row is
// the chain length -> page -> store, 3.7 us.

struct AppendArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* q_out;
    const uint16_t* q_weight;
    const uint16_t* k_weight;
    const float* inv_freq;
    uint8_t* k_pages;
    uint8_t* v_pages;
    const uint32_t* table;
    const uint32_t* lengths;
    const uint32_t* row_starts;
    uint32_t* error;
    uint64_t page_stride, head_stride;  // bytes
    uint32_t token_stride;              // bytes
    uint32_t q_stride, k_stride, v_stride, q_out_stride;
    uint32_t table_stride, num_seqs, rows, seq_rows, num_pages;
    uint32_t q_heads, kv_heads, dim, page_shift;
    uint32_t rot, normalize_v, weights16;
    uint32_t lanes_log2;  // lanes a head row takes, 16 elements each
    uint32_t groups, waves_per_row;
    float eps, k_inv_scale, v_inv_scale;
};

typedef float f4a4_t __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ void unpack8(uint4 u, float* y) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[2 * i] = f16_to_f32((uint16_t)(w[i] & 0xFFFFu));
        y[2 * i + 1] = f16_to_f32((uint16_t)(w[i] >> 16));
    }
}

__device__ __forceinline__ uint4 pack8_f16(const float* y) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = (uint32_t)f32_to_f16(y[2 * i]) | ((uint32_t)f32_to_f16(y[2 * i + 1]) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// x / scale clamped to e4m3's largest value, NaN kept.
__device__ __forceinline__ float e4m3_range(float x, float inv_scale) {
    const float y = x * inv_scale;
    return y > 448.0f ? 448.0f : (y < -448.0f ? -448.0f : y);
}

__device__ __forceinline__ uint2 pack8_e4m3(const float* y, float inv_scale) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int u = 0;
        u = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(y[4 * i], inv_scale),
                                            e4m3_range(y[4 * i + 1], inv_scale), u, false);
        u = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(y[4 * i + 2], inv_scale),
                                            e4m3_range(y[4 * i + 3], inv_scale), u, true);
        w[i] = (uint32_t)u;
    }
    return make_uint2(w[0], w[1]);
}

// A wave takes `groups` groups of one row's heads, 64 >> lanes_log2 heads each:
// queries, then keys, then values. Lane j of a head holds two 8-element chunks;
// for split pairs chunk j and chunk j + rot / 16, so that both elements of every
// pair are the lane's own, and its angles are inv_freq[8 j .. 8 j + 7] in either
// order of pairs, the same for all of the wave's heads.
template <bool E4M3, bool INTERLEAVED>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4u + (threadIdx.x >> 6));
    const uint32_t row = wave / a.waves_per_row;
    if (row >= a.rows) return;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t L = 1u << a.lanes_log2, j = lane & (L - 1u), per = 64u >> a.lanes_log2;
    const uint32_t heads = a.q_heads + 2u * a.kv_heads;
    const uint32_t chunks = a.dim / 8u, half = a.rot / 16u;
    const bool turns = j < half;
    const uint32_t q0 = !INTERLEAVED && turns ? j : 2u * j;  // the lane's chunks of q and k
    const uint32_t q1 = !INTERLEAVED && turns ? j + half : 2u * j + 1u;

    struct Head {
        uint32_t head, c0, c1;
        uint4 x0, x1;
    };
    const auto load = [&](uint32_t group) {
        Head t;
        t.head = group * per + (lane >> a.lanes_log2);
        const bool is_q = t.head < a.q_heads, is_v = t.head >= a.q_heads + a.kv_heads;
        t.c0 = is_v ? 2u * j : q0;
        t.c1 = is_v ? 2u * j + 1u : q1;
        const uint16_t* src =
            is_q   ? a.q + (uint64_t)row * a.q_stride + t.head * a.dim
            : is_v ? a.v + (uint64_t)row * a.v_stride + (t.head - a.q_heads - a.kv_heads) * a.dim
                   : a.k + (uint64_t)row * a.k_stride + (t.head - a.q_heads) * a.dim;
        t.x0 = t.x1 = make_uint4(0, 0, 0, 0);
        if (t.head < heads && t.c0 < chunks) t.x0 = *reinterpret_cast<const uint4*>(src + 8u * t.c0);
        if (t.head < heads && t.c1 < chunks) t.x1 = *reinterpret_cast<const uint4*>(src + 8u * t.c1);
        return t;
    };
    const uint32_t first = (wave % a.waves_per_row) * a.groups;
    const uint32_t all = (heads + per - 1u) / per;
    const uint32_t end = first + a.groups < all ? first + a.groups : all;
    Head next = load(first);

    // the norms' weights at the lane's chunks (8 bf16 each) and its frequencies
    const auto weights = [&](const uint16_t* w, uint32_t c) {
        if (!w || c >= chunks) return make_uint4(0, 0, 0, 0);
        if (a.weights16) return *reinterpret_cast<const uint4*>(w + 8u * c);
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            u[e] = (uint32_t)w[8u * c + 2 * e] | ((uint32_t)w[8u * c + 2 * e + 1] << 16);
        return make_uint4(u[0], u[1], u[2], u[3]);
    };
    const uint4 qw0 = weights(a.q_weight, q0), qw1 = weights(a.q_weight, q1);
    const uint4 kw0 = weights(a.k_weight, q0), kw1 = weights(a.k_weight, q1);
    f4a4_t f0 = {0, 0, 0, 0}, f1 = {0, 0, 0, 0};
    if (turns) {
        f0 = *reinterpret_cast<const f4a4_t*>(a.inv_freq + 8u * j);
        f1 = *reinterpret_cast<const f4a4_t*>(a.inv_freq + 8u * j + 4u);
    }

    bool broken;
    const uint32_t s =
        find_seq(a.row_starts, a.num_seqs, a.seq_rows, a.rows, row, a.error, &broken);
    if (s >= a.num_seqs && !broken) return;
    const uint32_t capacity = a.table_stride << a.page_shift;
    const SeqRows sr = broken ? SeqRows{0u, row, 1u, 0u, kErrAttnRows}
                              : seq_rows(a.row_starts, a.lengths, s, a.seq_rows, a.rows, capacity);
    const int32_t pos = (int32_t)sr.length - (int32_t)sr.count + (int32_t)(row - sr.first);
    bool drop = sr.bad || pos < 0;  // nothing to append; the query row becomes zeros (NaN)
    if (sr.bad && lane == 0) report(a.error, sr.bad);
    uint32_t page = 0;
    if (!drop) {
        page = scalar_load(a.table + ((uint64_t)s * a.table_stride + ((uint32_t)pos >> a.page_shift)));
        if (page >= a.num_pages) {
            drop = true;
            if (lane == 0) report(a.error, kErrAttnPage);
        }
    }
    const uint64_t slot = page * a.page_stride +
                          (uint64_t)((uint32_t)pos & ((1u << a.page_shift) - 1u)) * a.token_stride;

    float cs[8], sn[8];
    const double turn = (double)pos * 0.15915494309189535;  // 1 / 2 pi
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        double t = turn * (double)(e < 4 ? f0[e & 3] : f1[e & 3]);
        t -= __builtin_rint(t);
        cs[e] = __builtin_amdgcn_cosf((float)t);
        sn[e] = __builtin_amdgcn_sinf((float)t);
    }

    for (uint32_t group = first; group < end; ++group) {
        const Head t = next;
        if (group + 1u < end) next = load(group + 1u);
        const bool is_q = t.head < a.q_heads, is_v = t.head >= a.q_heads + a.kv_heads;
        float y[16];
        unpack8(t.x0, y);
        unpack8(t.x1, y + 8);
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) ss = __builtin_fmaf(y[e], y[e], ss);
        for (uint32_t o = L >> 1; o > 0; o >>= 1) ss += __shfl_xor(ss, (int)o, 64);
        if (is_v ? a.normalize_v != 0 : (is_q ? a.q_weight : a.k_weight) != nullptr) {
            const float inv = 1.0f / __builtin_sqrtf(ss / (float)a.dim + a.eps);
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] *= inv;
            if (!is_v) {
                const uint32_t w[8] = {is_q ? qw0.x : kw0.x, is_q ? qw0.y : kw0.y,
                                       is_q ? qw0.z : kw0.z, is_q ? qw0.w : kw0.w,
                                       is_q ? qw1.x : kw1.x, is_q ? qw1.y : kw1.y,
                                       is_q ? qw1.z : kw1.z, is_q ? qw1.w : kw1.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    y[2 * e] *= __uint_as_float(w[e] << 16);
                    y[2 * e + 1] *= __uint_as_float(w[e] & 0xFFFF0000u);
                }
            }
        }
        if (!is_v && turns) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = INTERLEAVED ? 2 * e : e, k = INTERLEAVED ? 2 * e + 1 : e + 8;
                const float u = y[i], w = y[k];
                y[i] = u * cs[e] - w * sn[e];
                y[k] = w * cs[e] + u * sn[e];
            }
        }
        if (t.head >= heads) continue;
        const bool has0 = t.c0 < chunks, has1 = t.c1 < chunks;
        if (is_q) {
            if (drop) {
                const float fill = pos < 0 && !sr.bad ? 0.0f : __builtin_nanf("");
#pragma unroll
                for (int e = 0; e < 16; ++e) y[e] = fill;
            }
            uint16_t* dst = a.q_out + (uint64_t)row * a.q_out_stride + t.head * a.dim;
            if (has0) *reinterpret_cast<uint4*>(dst + 8u * t.c0) = pack8_f16(y);
            if (has1) *reinterpret_cast<uint4*>(dst + 8u * t.c1) = pack8_f16(y + 8);
        } else if (!drop) {
            const uint32_t kvh = is_v ? t.head - a.q_heads - a.kv_heads : t.head - a.q_heads;
            uint8_t* dst = (is_v ? a.v_pages : a.k_pages) + slot + kvh * a.head_stride;
            if (E4M3) {
                const float inv_scale = is_v ? a.v_inv_scale : a.k_inv_scale;
                if (has0) *reinterpret_cast<uint2*>(dst + 8u * t.c0) = pack8_e4m3(y, inv_scale);
                if (has1) *reinterpret_cast<uint2*>(dst + 8u * t.c1) = pack8_e4m3(y + 8, inv_scale);
            } else {
                if (has0) *reinterpret_cast<uint4*>(dst + 16u * t.c0) = pack8_f16(y);
                if (has1) *reinterpret_cast<uint4*>(dst + 16u * t.c1) = pack8_f16(y + 8);
            }
        }
    }
}

}  // namespace
}  // namespace tsg

using namespace tsg;

extern "C" tsg_status tsg_attn_check(const tsg_attn_config* config, const tsg_kv_pages* pages,
                                     const tsg_attn_batch* batch) {
    if (tsg_status s = check_attn_config(config)) return s;
    if (pages)
        if (tsg_status s = check_attn_pages(*config, pages)) return s;
    if (batch)
        if (tsg_status s = check_attn_batch(*config, batch)) return s;
    return TSG_OK;
}

extern "C" tsg_status tsg_attn_create(tsg_ctx* ctx, const tsg_attn_config* config, tsg_attn** out) {
    TSG_REQUIRE(out, TSG_ERR_INVALID_ARGUMENT, "out is NULL");
    *out = nullptr;
    if (tsg_status s = check_attn_config(config)) return s;
    TSG_REQUIRE(ctx, TSG_ERR_INVALID_ARGUMENT, "ctx is NULL");
    tsg_attn* attn = new (std::nothrow) tsg_attn();
    TSG_REQUIRE(attn, TSG_ERR_OUT_OF_MEMORY, "host allocation failed");
    attn->ctx = ctx;
    attn->device = ctx->device;
    attn->cfg = *config;
    attn->group = config->q_heads / config->kv_heads;
    attn->page_shift = (uint32_t)__builtin_ctz(config->page_tokens);
    attn->cell = cell_bytes(*config);
    attn->padded_dim = 64u;
    while (attn->padded_dim < config->head_dim) attn->padded_dim *= 2u;
    DeviceScope scope(ctx->device);
    hipError_t e = scope.status;
    const size_t words = (size_t)kPartialRows * (attn->padded_dim + 2u);
    if (e == hipSuccess) e = hipMalloc(&attn->partials, words * sizeof(float));
    if (e == hipSuccess) e = hipMalloc(&attn->arrivals, kMaxPartials * sizeof(uint32_t));
    if (e == hipSuccess) e = hipMemset(attn->arrivals, 0, kMaxPartials * sizeof(uint32_t));
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        (void)hipFree(attn->partials);
        (void)hipFree(attn->arrivals);
        delete attn;
        return fail(TSG_ERR_OUT_OF_MEMORY, "attention scratch: %s", hipGetErrorString(e));
    }
    tsg_status s = prepare_decode(attn);
    if (s == TSG_OK) s = prepare_prefill(attn);
    if (s != TSG_OK) {
        (void)hipFree(attn->partials);
        (void)hipFree(attn->arrivals);
        delete attn;
        return s;
    }
    *out = attn;
    return TSG_OK;
}

extern "C" void tsg_attn_destroy(tsg_attn* attn) {
    if (!attn) return;
    DeviceScope scope(attn->device);
    (void)hipDeviceSynchronize();
    (void)hipFree(attn->partials);
    (void)hipFree(attn->arrivals);
    delete attn;
}

extern "C" tsg_status tsg_attn_append(tsg_attn* attn, tsg_stream stream, const tsg_kv_pages* pages,
                                      const tsg_attn_batch* batch, const tsg_attn_rows* rows,
                                      const tsg_attn_norm_rope* nr, uint16_t* q_out,
                                      uint32_t q_out_stride) {
    TSG_REQUIRE(attn, TSG_ERR_INVALID_ARGUMENT, "attn is NULL");
    const tsg_attn_config& c = attn->cfg;
    if (tsg_status s = check_attn_pages(c, pages)) return s;
    if (tsg_status s = check_attn_batch(c, batch)) return s;
    TSG_REQUIRE(pages->k != pages->v, TSG_ERR_INVALID_ARGUMENT,
                "append writes two pools: keys and values have one address");
    TSG_REQUIRE(rows && nr && rows->q && rows->k && rows->v && q_out, TSG_ERR_INVALID_ARGUMENT,
                "NULL append operand");
    const uint32_t q_width = c.q_heads * c.head_dim, kv_width = c.kv_heads * c.head_dim;
    TSG_REQUIRE(rows->q_stride >= q_width && q_out_stride >= q_width, TSG_ERR_INVALID_ARGUMENT,
                "q stride is too small");
    TSG_REQUIRE(rows->k_stride >= kv_width && rows->v_stride >= kv_width, TSG_ERR_INVALID_ARGUMENT,
                "k or v stride is too small");
    TSG_REQUIRE(is16(rows->q) && is16(rows->k) && is16(rows->v) && is16(q_out) &&
                    rows->q_stride % 8u == 0 && rows->k_stride % 8u == 0 &&
                    rows->v_stride % 8u == 0 && q_out_stride % 8u == 0,
                TSG_ERR_ALIGNMENT, "q, k and v rows must be 16-byte aligned");
    TSG_REQUIRE((rows->q == q_out && (rows->q_stride == q_out_stride || batch->rows == 1u)) ||
                    !rows_share(rows->q, rows->q_stride, q_width, q_out, q_out_stride, q_width,
                                batch->rows),
                TSG_ERR_INVALID_ARGUMENT, "q_out shares elements with q and is not q itself");
    TSG_REQUIRE(!rows_share(rows->k, rows->k_stride, kv_width, q_out, q_out_stride, q_width,
                            batch->rows) &&
                    !rows_share(rows->v, rows->v_stride, kv_width, q_out, q_out_stride, q_width,
                                batch->rows),
                TSG_ERR_INVALID_ARGUMENT, "q_out shares elements with k or v");
    TSG_REQUIRE(nr->rotary_dim <= c.head_dim && nr->rotary_dim % 16u == 0, TSG_ERR_UNSUPPORTED,
                "rotary_dim %u: a multiple of 16 up to head_dim", nr->rotary_dim);
    TSG_REQUIRE(nr->rotary_dim == 0 || nr->inv_freq, TSG_ERR_INVALID_ARGUMENT, "inv_freq is NULL");
    TSG_REQUIRE(is4(nr->inv_freq) && is2(nr->q_weight) && is2(nr->k_weight), TSG_ERR_ALIGNMENT,
                "norm weights must be 2-byte and inv_freq 4-byte aligned");
    TSG_REQUIRE(nr->eps >= 0.0f && std::isfinite(nr->eps), TSG_ERR_INVALID_ARGUMENT,
                "eps must be finite and not negative");
    AppendArgs a{};
    a.q = rows->q;
    a.k = rows->k;
    a.v = rows->v;
    a.q_out = q_out;
    a.q_weight = nr->q_weight;
    a.k_weight = nr->k_weight;
    a.inv_freq = nr->inv_freq;
    a.k_pages = static_cast<uint8_t*>(pages->k);
    a.v_pages = static_cast<uint8_t*>(pages->v);
    a.table = batch->page_table;
    a.lengths = batch->lengths;
    a.row_starts = batch->row_starts;
    a.error = attn->ctx->counters + kSyncErrorWord;
    a.page_stride = pages->page_stride * attn->cell;
    a.head_stride = pages->head_stride * attn->cell;
    a.token_stride = pages->token_stride * attn->cell;
    a.q_stride = rows->q_stride;
    a.k_stride = rows->k_stride;
    a.v_stride = rows->v_stride;
    a.q_out_stride = q_out_stride;
    a.table_stride = batch->table_stride;
    a.num_seqs = batch->num_seqs;
    a.rows = batch->rows;
    a.seq_rows = batch->row_starts ? 0u : batch->rows / batch->num_seqs;
    a.num_pages = pages->num_pages;
    a.q_heads = c.q_heads;
    a.kv_heads = c.kv_heads;
    a.dim = c.head_dim;
    a.page_shift = attn->page_shift;
    a.rot = nr->rotary_dim;
    a.weights16 = is16(nr->q_weight) && is16(nr->k_weight) ? 1u : 0u;
    a.normalize_v = nr->normalize_v ? 1u : 0u;
    while ((16u << a.lanes_log2) < c.head_dim) ++a.lanes_log2;
    const uint32_t heads = c.q_heads + 2u * c.kv_heads, per_wave = 64u >> a.lanes_log2;
    // A wave takes all of a row (its sequence, page and angles found once) when
    // the rows alone give every SIMD eight waves; few rows spread out.
    const uint32_t groups = (heads + per_wave - 1u) / per_wave;
    const uint32_t spread = 32u * (uint32_t)attn->ctx->num_cus / a.rows;
    a.groups = spread >= groups ? 1u : groups / (spread > 1u ? spread : 1u);
    a.waves_per_row = (groups + a.groups - 1u) / a.groups;
    a.eps = nr->eps;
    a.k_inv_scale = 1.0f / c.k_scale;
    a.v_inv_scale = 1.0f / c.v_scale;
    DeviceScope scope(attn->device);
    TSG_HIP_TRY(scope.status);
    const uint64_t waves = (uint64_t)a.rows * a.waves_per_row;
    TSG_REQUIRE((waves + 3u) / 4u <= kMaxBlocks, TSG_ERR_UNSUPPORTED, "too many rows and heads for one launch");
    const dim3 grid((uint32_t)((waves + 3u) / 4u));
    const bool e4m3 = c.kv_type == TSG_KV_E4M3;
    const auto kernel = nr->interleaved ? (e4m3 ? append_kernel<true, true> : append_kernel<false, true>)
                                        : (e4m3 ? append_kernel<true, false> : append_kernel<false, false>);
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, as_stream(stream), a);
    return check_launch("attn_append");
}

extern "C" tsg_status tsg_attn_decode(tsg_attn* attn, tsg_stream stream, const tsg_kv_pages* pages,
                                      const tsg_attn_batch* batch, const uint16_t* q,
                                      uint32_t q_stride, uint16_t* out, uint32_t out_stride) {
    AttnArgs a{};
    if (tsg_status s = attn_args(attn, pages, batch, q, q_stride, out, out_stride, &a)) return s;
    TSG_REQUIRE(!batch->row_starts, TSG_ERR_INVALID_ARGUMENT,
                "decode takes the same 1...%u rows of every sequence (no row starts)",
                kMaxDecodeRows);
    TSG_REQUIRE(a.seq_rows <= kMaxDecodeRows, TSG_ERR_DECLINED,
                "more than %u rows a sequence: tsg_attn_prefill", kMaxDecodeRows);
    DeviceScope scope(attn->device);
    TSG_HIP_TRY(scope.status);
    return launch_decode(attn, a, stream);
}

// Few rows of wide heads, and so few tiles of them that most of the card would
// idle: the decode kernel splits the keys finer. One sequence, heads of 512 (16
// query, 2 key heads), decode against prefill kernel: 32 rows of the group over 4000
// keys 36 and 39 us, 256 rows 42 and 50, 32 over 32,000 keys 84 and 192, 256 162 and
// 163, but 512 rows 667 and 175; heads of 256 (16, 8): 8 rows over 4000 keys 18
// and 24, 64 rows 26 and 29, over 32,000 62 and 73, 73 and 74, but 256 rows 181
// and 110. More sequences, heads of 512, 32 rows over 32,000 keys: 4 (16 tiles) 123 and
// 161, 16 (64) 401 and 442; 256 rows: 4 (128) 670 and 268. Heads of 256: 4 of 8 rows
// (32) 196 and 197, 4 of 64 (128) 321 and 205, 16 of 8 (128) 694 and 701, over 1000
// keys 29 and 31. Narrower heads gain only under about 1000 keys (10 and 13) and lose
// beyond.
static bool decode_takes(const tsg_attn* attn, const AttnArgs& a) {
    if (a.row_starts || attn->padded_dim < 256u) return false;
    const uint64_t rows = (uint64_t)a.seq_rows * a.group;
    const uint64_t tiles =
        a.num_seqs * (uint64_t)a.kv_heads * ((rows + kDecodeTileRows - 1u) / kDecodeTileRows);
    return rows <= (attn->padded_dim == 256u ? 64u : 256u) &&
           tiles <= (uint64_t)attn->ctx->num_cus / 4u;
}

extern "C" tsg_status tsg_attn_prefill(tsg_attn* attn, tsg_stream stream,
                                       const tsg_kv_pages* pages, const tsg_attn_batch* batch,
                                       const uint16_t* q, uint32_t q_stride, uint16_t* out,
                                       uint32_t out_stride) {
    AttnArgs a{};
    if (tsg_status s = attn_args(attn, pages, batch, q, q_stride, out, out_stride, &a)) return s;
    DeviceScope scope(attn->device);
    TSG_HIP_TRY(scope.status);
    return decode_takes(attn, a) ? launch_decode(attn, a, stream) : launch_prefill(attn, a, stream);
}

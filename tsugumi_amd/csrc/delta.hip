// delta.hip — the gated delta rule's plan and checks, the causal convolution
// before it, and the rule row by row.
#include "delta_internal.hpp"

#include <cmath>
#include <new>

namespace tsg {
namespace {

constexpr uint32_t kMaxValueHeads = 256, kMaxKeyDim = 256, kMaxValueDim = 512;
constexpr uint32_t kMinConv = 2, kMaxConv = 8;
constexpr uint32_t kMaxDeltaSeqs = 1u << 16;
constexpr uint32_t kMaxDeltaRows = 1u << 22;
constexpr uint32_t kMaxStride = 1u << 27;

bool is16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool is4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
bool is2(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1u) == 0; }

uint32_t channels_of(const tsg_delta_config& c) {
    return 2u * c.key_heads * c.key_dim + c.value_heads * c.value_dim;
}

tsg_status check_config(const tsg_delta_config* c) {
    TSG_REQUIRE(c, TSG_ERR_INVALID_ARGUMENT, "delta config is NULL");
    TSG_REQUIRE(c->key_heads > 0 && c->value_heads > 0 && c->value_heads <= kMaxValueHeads,
                TSG_ERR_INVALID_ARGUMENT, "head counts must be in 1...%u", kMaxValueHeads);
    TSG_REQUIRE(c->value_heads % c->key_heads == 0, TSG_ERR_INVALID_ARGUMENT,
                "%u value heads do not share %u key heads evenly", c->value_heads, c->key_heads);
    TSG_REQUIRE(c->key_dim > 0 && c->key_dim <= kMaxKeyDim && c->key_dim % 16u == 0,
                TSG_ERR_UNSUPPORTED, "key_dim %u: a multiple of 16 up to %u", c->key_dim,
                kMaxKeyDim);
    TSG_REQUIRE(c->value_dim > 0 && c->value_dim <= kMaxValueDim && c->value_dim % 16u == 0,
                TSG_ERR_UNSUPPORTED, "value_dim %u: a multiple of 16 up to %u", c->value_dim,
                kMaxValueDim);
    TSG_REQUIRE(c->conv_width >= kMinConv && c->conv_width <= kMaxConv, TSG_ERR_UNSUPPORTED,
                "conv_width %u: %u...%u", c->conv_width, kMinConv, kMaxConv);
    TSG_REQUIRE(std::isfinite(c->scale) && std::fabs(c->scale) <= 1e6f, TSG_ERR_INVALID_ARGUMENT,
                "scale must be finite and at most 1e6");
    TSG_REQUIRE(c->eps >= 1e-12f && c->eps <= 1.0f, TSG_ERR_INVALID_ARGUMENT,
                "eps must be in 1e-12...1");
    return TSG_OK;
}

tsg_status check_states(const tsg_delta_config& c, const tsg_delta_states* p) {
    TSG_REQUIRE(p, TSG_ERR_INVALID_ARGUMENT, "delta states are NULL");
    TSG_REQUIRE(p->num_slots > 0 && p->num_slots < TSG_NO_SLOT, TSG_ERR_INVALID_ARGUMENT,
                "a pool needs at least one slot");
    TSG_REQUIRE(is16(p->s) && is16(p->conv), TSG_ERR_ALIGNMENT, "state pools must be 16-byte aligned");
    TSG_REQUIRE(p->slot_stride % 4u == 0 && p->conv_stride % 8u == 0, TSG_ERR_ALIGNMENT,
                "slot strides must be multiples of 16 bytes");
    const uint64_t slot = (uint64_t)c.value_heads * c.key_dim * c.value_dim;
    const uint64_t conv = (uint64_t)(c.conv_width - 1u) * channels_of(c);
    TSG_REQUIRE(!p->s || p->num_slots == 1u || p->slot_stride >= slot, TSG_ERR_INVALID_ARGUMENT,
                "slot stride is too small: states overlap");
    TSG_REQUIRE(!p->conv || p->num_slots == 1u || p->conv_stride >= conv, TSG_ERR_INVALID_ARGUMENT,
                "convolution stride is too small: states overlap");
    // with up to 2^32 slots every byte offset stays under 2^63
    TSG_REQUIRE(p->slot_stride < (1ull << 28) && p->conv_stride < (1ull << 28),
                TSG_ERR_INVALID_ARGUMENT, "slot stride too large");
    return TSG_OK;
}

tsg_status check_batch(const tsg_delta_batch* b) {
    TSG_REQUIRE(b, TSG_ERR_INVALID_ARGUMENT, "delta batch is NULL");
    TSG_REQUIRE(b->num_seqs > 0 && b->num_seqs <= kMaxDeltaSeqs, TSG_ERR_INVALID_ARGUMENT,
                "numSeqs must be in 1...%u", kMaxDeltaSeqs);
    TSG_REQUIRE(b->rows > 0 && b->rows <= kMaxDeltaRows, TSG_ERR_INVALID_ARGUMENT,
                "rows must be in 1...%u", kMaxDeltaRows);
    TSG_REQUIRE(b->in_slots && b->out_slots, TSG_ERR_INVALID_ARGUMENT, "NULL in or out slots");
    TSG_REQUIRE(is4(b->in_slots) && is4(b->out_slots) && is4(b->row_starts), TSG_ERR_ALIGNMENT,
                "slots and row starts must be 4-byte aligned");
    TSG_REQUIRE(b->row_starts || b->rows % b->num_seqs == 0, TSG_ERR_INVALID_ARGUMENT,
                "%u rows do not divide over %u sequences (give row starts)", b->rows, b->num_seqs);
    TSG_REQUIRE(b->kept == 1u || (!b->row_starts && b->kept <= kMaxDeltaKept &&
                                  b->kept == b->rows / b->num_seqs),
                TSG_ERR_INVALID_ARGUMENT,
                "kept is 1 or, of up to %u rows of every sequence, their number", kMaxDeltaKept);
    return TSG_OK;
}

tsg_status check_rows(const tsg_delta_config& c, const tsg_delta_rows* r) {
    TSG_REQUIRE(r && r->q && r->k && r->v && r->a && r->b, TSG_ERR_INVALID_ARGUMENT,
                "NULL delta rows");
    const uint32_t kw = c.key_heads * c.key_dim, vw = c.value_heads * c.value_dim;
    TSG_REQUIRE(r->q_stride >= kw && r->k_stride >= kw && r->v_stride >= vw,
                TSG_ERR_INVALID_ARGUMENT, "q, k or v stride is too small");
    TSG_REQUIRE(r->a_stride >= c.value_heads && r->b_stride >= c.value_heads,
                TSG_ERR_INVALID_ARGUMENT, "a or b stride is too small");
    // 16 rows are addressed by 32-bit byte offsets
    TSG_REQUIRE(r->q_stride <= kMaxStride && r->k_stride <= kMaxStride && r->v_stride <= kMaxStride,
                TSG_ERR_UNSUPPORTED, "row strides must be at most %u elements", kMaxStride);
    TSG_REQUIRE(is16(r->q) && is16(r->k) && is16(r->v) && r->q_stride % 8u == 0 &&
                    r->k_stride % 8u == 0 && r->v_stride % 8u == 0,
                TSG_ERR_ALIGNMENT, "q, k and v rows must be 16-byte aligned");
    TSG_REQUIRE(is2(r->a) && is2(r->b), TSG_ERR_ALIGNMENT, "a and b must be 2-byte aligned");
    return TSG_OK;
}

// Whether rows of `a` may share an element with rows of `b`: of one stride, the places
// within it; of two, their whole extents.
bool may_share(const uint16_t* a, uint64_t a_stride, uint64_t a_width, const uint16_t* b,
               uint64_t b_stride, uint64_t b_width, uint64_t rows) {
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
    const uint64_t a_bytes = 2u * ((rows - 1u) * a_stride + a_width);
    const uint64_t b_bytes = 2u * ((rows - 1u) * b_stride + b_width);
    if (pa + a_bytes <= pb || pb + b_bytes <= pa) return false;
    if (rows == 1u || a_stride != b_stride) return true;
    const uint64_t stride = 2u * a_stride;
    const bool a_first = pa <= pb;
    const uint64_t off = (a_first ? pb - pa : pa - pb) % stride;
    return off < 2u * (a_first ? a_width : b_width) ||
           off + 2u * (a_first ? b_width : a_width) > stride;
}

void fill_seqs(const tsg_delta* delta, const tsg_delta_states* states, const tsg_delta_batch* b,
               DeltaSeqs* d) {
    d->row_starts = b->row_starts;
    d->in_slots = b->in_slots;
    d->out_slots = b->out_slots;
    d->error = delta->ctx->counters + kSyncErrorWord;
    d->num_seqs = b->num_seqs;
    d->rows = b->rows;
    d->seq_rows = b->row_starts ? 0u : b->rows / b->num_seqs;
    d->kept = b->kept;
    d->num_slots = states->num_slots;
}

// ------------------------------------------------------------- convolution
//
// y[t, c] = silu(sum_j w[c, j] x[t - W + 1 + j, c]). Elementwise over the channels, so HBM
// bounds a prompt: a thread takes 8 channels (16 bytes) of up to 16 rows, all of
// whose loads go out together, and reads the W - 1 rows before them again (from L2).
// The thread with a sequence's first rows also moves its state, which it alone
// reads and writes, so one slot may be both in and out. 11207 rows of 8192 channels 76 us
// (4.85 TB/s); a token 4.3 us.

constexpr uint32_t kConvRows = 16;

struct ConvArgs {
    DeltaSeqs seqs;
    const uint16_t* x;
    const uint16_t* weight;
    uint16_t* out;
    uint16_t* states;
    uint64_t slot_stride;
    uint32_t x_stride, out_stride, channels;
    uint32_t pieces;  // workgroups across the channels
};

__device__ __forceinline__ void unpack8(uint4 u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = f16_to_f32((uint16_t)w[i]);
        f[2 * i + 1] = f16_to_f32((uint16_t)(w[i] >> 16));
    }
}

template <uint32_t W>
__global__ __launch_bounds__(256) void conv_kernel(ConvArgs p) {
    const DeltaSeqs& d = p.seqs;
    const DeltaTile t = delta_tile<kConvRows>(d, blockIdx.x / p.pieces);
    if (t.kind == 0u) return;
    const uint32_t piece = blockIdx.x % p.pieces, c0 = (piece * blockDim.x + threadIdx.x) * 8u;
    const bool live = c0 < p.channels;
    const uint4 nan8 = make_uint4(kDeltaNan2, kDeltaNan2, kDeltaNan2, kDeltaNan2);
    if (t.kind == 2u) {
        if (live)
            for (uint32_t r = t.first; r < t.first + t.count; ++r)
                *reinterpret_cast<uint4*>(p.out + (uint64_t)r * p.out_stride + c0) = nan8;
        if (blockIdx.x == 0 && threadIdx.x == 0) report(d.error, kErrDeltaRows);
        return;
    }
    const DeltaSeq q = delta_seq(d, t.seq);
    const bool bad = out_slots_clash(d, t.seq) || q.bad;
    if (bad && t.tile == 0u && piece == 0u && threadIdx.x == 0) report(d.error, kErrDeltaSlot);
    if (!live) return;
    const uint16_t* x = p.x + c0;
    uint16_t* out = p.out + c0;
    if (bad) {
        for (uint32_t r = t.first; r < t.first + t.count; ++r)
            *reinterpret_cast<uint4*>(out + (uint64_t)r * p.out_stride) = nan8;
        return;
    }
    // inputs W - 1 before the tile's first row, and its rows
    uint4 in[kConvRows + W - 1u];
    const uint16_t* old = p.states + (uint64_t)q.in * p.slot_stride + c0;
    const auto before = [&](uint32_t j) -> uint4 {  // input j of the state
        if (q.fresh) return make_uint4(0, 0, 0, 0);
        return *reinterpret_cast<const uint4*>(old + (uint64_t)j * p.channels);
    };
    const bool first = t.tile == 0u;
#pragma unroll
    for (uint32_t i = 0; i < W - 1u; ++i)
        in[i] = first ? before(i) : *reinterpret_cast<const uint4*>(
                                        x + (uint64_t)(t.first - (W - 1u) + i) * p.x_stride);
#pragma unroll
    for (uint32_t i = 0; i < kConvRows; ++i)
        in[W - 1u + i] = i < t.count ? *reinterpret_cast<const uint4*>(
                                           x + (uint64_t)(t.first + i) * p.x_stride)
                                     : make_uint4(0, 0, 0, 0);
    uint4 wbits[W];  // [8 channels][W] bf16
#pragma unroll
    for (uint32_t j = 0; j < W; ++j)
        wbits[j] = *reinterpret_cast<const uint4*>(p.weight + (uint64_t)c0 * W + 8u * j);
    const auto weight = [&](uint32_t c, uint32_t j) {
        const uint32_t n = c * W + j;
        const uint4 u = wbits[n / 8u];
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        return bf16_to_f32((uint16_t)(w[n % 8u / 2u] >> (16u * (n % 2u))));
    };

    // the state behind row n - 1 (of the sequence): its last W - 1 inputs
    const auto keep = [&](uint32_t n, uint32_t slot) {
        if (slot == TSG_NO_SLOT) return;
        uint16_t* to = p.states + (uint64_t)slot * p.slot_stride + c0;
        uint4 u[W - 1u];
#pragma unroll
        for (uint32_t j = 0; j < W - 1u; ++j) {
            const uint32_t at = n + j;  // counted from the old state's first input
            if (at < W - 1u) {
                u[j] = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (uint32_t i = 0; i < W - 1u; ++i)
                    if (i == at) u[j] = in[i];
                // else the compiler loads one of two addresses here, and `in` goes to memory
                asm("" : "+v"(u[j].x), "+v"(u[j].y), "+v"(u[j].z), "+v"(u[j].w));
            } else {
                u[j] = *reinterpret_cast<const uint4*>(
                    x + (uint64_t)(q.first + at - (W - 1u)) * p.x_stride);
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < W - 1u; ++j)
            *reinterpret_cast<uint4*>(to + (uint64_t)j * p.channels) = u[j];
    };
    if (first) {
        if (d.kept == 1u)
            keep(q.count, scalar_load(d.out_slots + t.seq));
        else
            for (uint32_t i = 0; i < d.kept; ++i)
                keep(i + 1u, scalar_load(d.out_slots + t.seq * d.kept + i));
    }

    float win[W][8];  // the last W inputs, input i in place i % W
#pragma unroll
    for (uint32_t i = 0; i < W - 1u; ++i) unpack8(in[i], win[i]);
#pragma unroll
    for (uint32_t i = 0; i < kConvRows; ++i) {
        if (i >= t.count) continue;
        unpack8(in[W - 1u + i], win[(W - 1u + i) % W]);
        uint32_t h[4];
#pragma unroll
        for (uint32_t c = 0; c < 8u; ++c) {
            float y = 0.0f;
#pragma unroll
            for (uint32_t j = 0; j < W; ++j) y = __builtin_fmaf(weight(c, j), win[(i + j) % W][c], y);
            // y / (1 + e^-y)
            const float e = __builtin_amdgcn_exp2f(y * -1.4426950408889634f);
            const uint32_t bits = f32_to_f16(y * __builtin_amdgcn_rcpf(1.0f + e));
            h[c / 2u] = c % 2u ? h[c / 2u] | bits << 16 : bits;
        }
        *reinterpret_cast<uint4*>(out + (uint64_t)(t.first + i) * p.out_stride) =
            make_uint4(h[0], h[1], h[2], h[3]);
    }
}

// ------------------------------------------------------------- row by row
//
// S <- e S; u = beta (v - S^T k); S <- S + k u^T; o = S^T q. With both products of
// the state before the row, o = e S^T q + (q . k) u needs one sum over the key
// elements a row, and the state stays in registers: a wave takes 32 of a head's
// value elements (128-byte pieces of the state's rows), a lane four of them and
// an eighth of the key elements. Every state is read and written once: HBM bounds
// a batch, latency one sequence (64 states of 32 heads of 128 x 128 58 us, 4.7 TB/s; one 6 us).

template <uint32_t DKP>
__global__ __launch_bounds__(256) void recurrent_kernel(DeltaArgs p) {
    constexpr uint32_t R = DKP / 8u;  // key elements of a lane
    const DeltaSeqs& d = p.seqs;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t slices = (p.value_dim + 31u) / 32u;
    const uint32_t id = blockIdx.x * (blockDim.x >> 6) +
                        __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t head = id / slices % p.value_heads, s = id / slices / p.value_heads;
    if (s >= d.num_seqs) return;
    const uint32_t c = id % slices * 32u + 4u * (lane & 7u), r0 = (lane >> 3) * R;
    const bool c_in = c < p.value_dim;
    const uint32_t vc = head * p.value_dim + c;
    const DeltaSlot sq = delta_slot(d, s);
    const uint32_t first = s * d.seq_rows;
    const uint64_t place = (uint64_t)head * p.key_dim * p.value_dim + (uint64_t)r0 * p.value_dim + c;
    // key_dim is a multiple of 16: eight rows are in or out together
    const auto in8 = [&](uint32_t i) { return c_in && r0 + (i & ~7u) < p.key_dim; };
    f4_t st[R];
#pragma unroll
    for (uint32_t i = 0; i < R; ++i) {
        st[i] = f4_t{0, 0, 0, 0};
        if (!sq.fresh && in8(i))
            st[i] = *reinterpret_cast<const f4_t*>(p.s + (uint64_t)sq.in * p.slot_stride + place +
                                                   i * p.value_dim);
    }
    const bool bad = out_slots_clash(d, s) || sq.bad;
    if (bad && lane == 0u && id % slices == 0u && head == 0u) report(d.error, kErrDeltaSlot);

    const uint32_t kh = head / p.group * p.key_dim + r0;
    const float rate = expf(p.a_log[head]), bias = p.dt_bias[head];
    const auto load_key = [&](const uint16_t* row, uint4 (&u)[R / 8u]) {
#pragma unroll
        for (uint32_t i = 0; i < R / 8u; ++i)
            u[i] = r0 + 8u * i < p.key_dim ? *reinterpret_cast<const uint4*>(row + kh + 8u * i)
                                           : make_uint4(0, 0, 0, 0);
    };
    const auto store = [&](uint32_t slot) {
        if (slot == TSG_NO_SLOT || bad) return;
        float* to = p.s + (uint64_t)slot * p.slot_stride + place;
#pragma unroll
        for (uint32_t i = 0; i < R; ++i)
            if (in8(i)) *reinterpret_cast<f4_t*>(to + i * p.value_dim) = st[i];
    };
    uint4 qn[R / 8u], kn[R / 8u];
    uint2 vn = make_uint2(0, 0);
    uint32_t an = 0, bn = 0;
    const auto fetch = [&](uint32_t i) {
        const uint64_t row = first + i;
        load_key(p.q + row * p.q_stride, qn);
        load_key(p.k + row * p.k_stride, kn);
        if (c_in) vn = *reinterpret_cast<const uint2*>(p.v + row * p.v_stride + vc);
        an = p.a[row * p.a_stride + head];
        bn = p.b[row * p.b_stride + head];
    };
    fetch(0u);
#pragma unroll 1
    for (uint32_t row = 0; row < d.seq_rows; ++row) {
        float q[R], k[R];
#pragma unroll
        for (uint32_t i = 0; i < R; i += 8u) {
            float f[8];
            unpack8(qn[i / 8u], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) q[i + e] = f[e];
            unpack8(kn[i / 8u], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) k[i + e] = f[e];
        }
        const uint2 vb = vn;
        const float av = f16_to_f32((uint16_t)an) + bias, bv = f16_to_f32((uint16_t)bn);
        if (row + 1u < d.seq_rows) fetch(row + 1u);
        // sums over the key elements: |q|^2, |k|^2, q . k, S^T k, S^T q
        float sum[11];
#pragma unroll
        for (int e = 0; e < 11; ++e) sum[e] = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < R; ++i) {
            sum[0] = __builtin_fmaf(q[i], q[i], sum[0]);
            sum[1] = __builtin_fmaf(k[i], k[i], sum[1]);
            sum[2] = __builtin_fmaf(q[i], k[i], sum[2]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sum[3 + e] = __builtin_fmaf(st[i][e], k[i], sum[3 + e]);
                sum[7 + e] = __builtin_fmaf(st[i][e], q[i], sum[7 + e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 11; ++e)
            sum[e] = sum_across32(sum_across16(sum[e] + dpp_f32<0x128>(sum[e])));
        const float rq = p.scale / sqrtf(sum[0] + p.eps), rk = 1.0f / sqrtf(sum[1] + p.eps);
        const float soft = fmaxf(av, 0.0f) + log1pf(expf(-fabsf(av)));
        const float decay = av != av ? av : expf(-rate * soft);
        const float beta = 1.0f / (1.0f + expf(-bv));
        const float v[4] = {f16_to_f32((uint16_t)vb.x), f16_to_f32((uint16_t)(vb.x >> 16)),
                            f16_to_f32((uint16_t)vb.y), f16_to_f32((uint16_t)(vb.y >> 16))};
        float u[4], o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            u[e] = beta * (v[e] - decay * rk * sum[3 + e]);
            o[e] = decay * rq * sum[7 + e] + rq * rk * sum[2] * u[e];
            u[e] *= rk;
        }
#pragma unroll
        for (uint32_t i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) st[i][e] = __builtin_fmaf(k[i], u[e], decay * st[i][e]);
        if (lane < 8u && c_in) {
            uint2 h = make_uint2((uint32_t)f32_to_f16(o[0]) | (uint32_t)f32_to_f16(o[1]) << 16,
                                 (uint32_t)f32_to_f16(o[2]) | (uint32_t)f32_to_f16(o[3]) << 16);
            if (bad) h = make_uint2(kDeltaNan2, kDeltaNan2);
            *reinterpret_cast<uint2*>(p.out + (uint64_t)(first + row) * p.out_stride + vc) = h;
        }
        if (d.kept > 1u) store(scalar_load(d.out_slots + s * d.kept + row));
    }
    if (d.kept == 1u) store(scalar_load(d.out_slots + s));
}

tsg_status delta_args(const tsg_delta* delta, const tsg_delta_states* states,
                      const tsg_delta_batch* batch, const tsg_delta_rows* rows, const float* a_log,
                      const float* dt_bias, uint16_t* out, uint32_t out_stride, DeltaArgs* a) {
    TSG_REQUIRE(delta, TSG_ERR_INVALID_ARGUMENT, "delta is NULL");
    const tsg_delta_config& c = delta->cfg;
    if (tsg_status s = check_states(c, states)) return s;
    if (tsg_status s = check_batch(batch)) return s;
    if (tsg_status s = check_rows(c, rows)) return s;
    TSG_REQUIRE(states->s, TSG_ERR_INVALID_ARGUMENT, "the states' pool is NULL");
    TSG_REQUIRE(a_log && dt_bias && out, TSG_ERR_INVALID_ARGUMENT, "NULL delta operand");
    TSG_REQUIRE(is4(a_log) && is4(dt_bias), TSG_ERR_ALIGNMENT,
                "a_log and dt_bias must be 4-byte aligned");
    const uint32_t kw = c.key_heads * c.key_dim, vw = c.value_heads * c.value_dim;
    TSG_REQUIRE(out_stride >= vw, TSG_ERR_INVALID_ARGUMENT, "out stride is too small");
    TSG_REQUIRE(out_stride <= kMaxStride, TSG_ERR_UNSUPPORTED,
                "row strides must be at most %u elements", kMaxStride);
    TSG_REQUIRE(is16(out) && out_stride % 8u == 0, TSG_ERR_ALIGNMENT,
                "out rows must be 16-byte aligned");
    const struct {
        const uint16_t* p;
        uint32_t stride, width;
    } ins[] = {{rows->q, rows->q_stride, kw},
               {rows->k, rows->k_stride, kw},
               {rows->v, rows->v_stride, vw},
               {rows->a, rows->a_stride, c.value_heads},
               {rows->b, rows->b_stride, c.value_heads}};
    for (const auto& r : ins)
        TSG_REQUIRE(!may_share(r.p, r.stride, r.width, out, out_stride, vw, batch->rows),
                    TSG_ERR_INVALID_ARGUMENT, "out shares elements with the rows");
    fill_seqs(delta, states, batch, &a->seqs);
    a->q = rows->q;
    a->k = rows->k;
    a->v = rows->v;
    a->a = rows->a;
    a->b = rows->b;
    a->a_log = a_log;
    a->dt_bias = dt_bias;
    a->out = out;
    a->s = states->s;
    a->slot_stride = states->slot_stride;
    a->q_stride = rows->q_stride;
    a->k_stride = rows->k_stride;
    a->v_stride = rows->v_stride;
    a->a_stride = rows->a_stride;
    a->b_stride = rows->b_stride;
    a->out_stride = out_stride;
    a->value_heads = c.value_heads;
    a->group = delta->group;
    a->key_dim = c.key_dim;
    a->value_dim = c.value_dim;
    a->scale = c.scale;
    a->eps = c.eps;
    return TSG_OK;
}

tsg_status launch_recurrent(const tsg_delta* delta, const DeltaArgs& a, tsg_stream stream) {
    const uint64_t waves =
        (uint64_t)a.seqs.num_seqs * a.value_heads * ((a.value_dim + 31u) / 32u);
    // few waves: one a workgroup, so that they spread over the CUs
    const uint32_t per = waves <= 4u * (uint64_t)delta->ctx->num_cus ? 1u : 4u;
    const dim3 grid((uint32_t)((waves + per - 1u) / per)), block(64u * per);
    TSG_REQUIRE((waves + per - 1u) / per <= kMaxBlocks, TSG_ERR_UNSUPPORTED,
                "too many sequences and heads for one launch");
    const auto kernel = delta->padded_key == 64u    ? recurrent_kernel<64>
                        : delta->padded_key == 128u ? recurrent_kernel<128>
                                                    : recurrent_kernel<256>;
    hipLaunchKernelGGL(kernel, grid, block, 0, as_stream(stream), a);
    return check_launch("delta_recurrent");
}

}  // namespace
}  // namespace tsg

using namespace tsg;

extern "C" tsg_status tsg_delta_check(const tsg_delta_config* config,
                                      const tsg_delta_states* states,
                                      const tsg_delta_batch* batch, const tsg_delta_rows* rows) {
    if (tsg_status s = check_config(config)) return s;
    if (states)
        if (tsg_status s = check_states(*config, states)) return s;
    if (batch)
        if (tsg_status s = check_batch(batch)) return s;
    if (rows)
        if (tsg_status s = check_rows(*config, rows)) return s;
    return TSG_OK;
}

extern "C" tsg_status tsg_delta_create(tsg_ctx* ctx, const tsg_delta_config* config,
                                       tsg_delta** out) {
    TSG_REQUIRE(out, TSG_ERR_INVALID_ARGUMENT, "out is NULL");
    *out = nullptr;
    if (tsg_status s = check_config(config)) return s;
    TSG_REQUIRE(ctx, TSG_ERR_INVALID_ARGUMENT, "ctx is NULL");
    tsg_delta* delta = new (std::nothrow) tsg_delta();
    TSG_REQUIRE(delta, TSG_ERR_OUT_OF_MEMORY, "host allocation failed");
    delta->ctx = ctx;
    delta->device = ctx->device;
    delta->cfg = *config;
    delta->group = config->value_heads / config->key_heads;
    delta->channels = channels_of(*config);
    delta->padded_key = config->key_dim <= 64u ? 64u : config->key_dim <= 128u ? 128u : 256u;
    DeviceScope scope(ctx->device);
    tsg_status s = scope.status == hipSuccess
                       ? prepare_delta(delta)
                       : fail(TSG_ERR_HIP, "device: %s", hipGetErrorString(scope.status));
    if (s != TSG_OK) {
        delete delta;
        return s;
    }
    *out = delta;
    return TSG_OK;
}

extern "C" void tsg_delta_destroy(tsg_delta* delta) { delete delta; }

extern "C" tsg_status tsg_delta_conv(tsg_delta* delta, tsg_stream stream,
                                     const tsg_delta_states* states, const tsg_delta_batch* batch,
                                     const uint16_t* x, uint32_t x_stride, const uint16_t* weight,
                                     uint16_t* out, uint32_t out_stride) {
    TSG_REQUIRE(delta, TSG_ERR_INVALID_ARGUMENT, "delta is NULL");
    if (tsg_status s = check_states(delta->cfg, states)) return s;
    if (tsg_status s = check_batch(batch)) return s;
    TSG_REQUIRE(states->conv, TSG_ERR_INVALID_ARGUMENT, "the convolution's pool is NULL");
    TSG_REQUIRE(x && weight && out, TSG_ERR_INVALID_ARGUMENT, "NULL convolution operand");
    TSG_REQUIRE(x_stride >= delta->channels && out_stride >= delta->channels,
                TSG_ERR_INVALID_ARGUMENT, "x or out stride is too small");
    TSG_REQUIRE(is16(x) && is16(out) && is16(weight) && x_stride % 8u == 0 && out_stride % 8u == 0,
                TSG_ERR_ALIGNMENT, "x and out rows and the weight must be 16-byte aligned");
    TSG_REQUIRE(!may_share(x, x_stride, delta->channels, out, out_stride, delta->channels,
                           batch->rows),
                TSG_ERR_INVALID_ARGUMENT, "out shares elements with x");
    ConvArgs a{};
    fill_seqs(delta, states, batch, &a.seqs);
    a.x = x;
    a.weight = weight;
    a.out = out;
    a.states = states->conv;
    a.slot_stride = states->conv_stride;
    a.x_stride = x_stride;
    a.out_stride = out_stride;
    a.channels = delta->channels;
    const uint32_t tiles =
        delta_tiles<kConvRows>(batch->rows, batch->num_seqs, a.seqs.seq_rows, batch->row_starts);
    const uint32_t lanes = delta->channels / 8u;
    // few rows: one wave a workgroup, so that they spread over the CUs
    const uint32_t threads = (uint64_t)tiles * lanes <= 256u * (uint64_t)delta->ctx->num_cus ? 64u : 256u;
    a.pieces = (lanes + threads - 1u) / threads;
    TSG_REQUIRE((uint64_t)a.pieces * tiles <= kMaxBlocks, TSG_ERR_UNSUPPORTED,
                "too many rows and channels for one launch");
    DeviceScope scope(delta->device);
    TSG_HIP_TRY(scope.status);
    static constexpr void (*kKernels[])(ConvArgs) = {conv_kernel<2>, conv_kernel<3>, conv_kernel<4>,
                                                     conv_kernel<5>, conv_kernel<6>, conv_kernel<7>,
                                                     conv_kernel<8>};
    hipLaunchKernelGGL(kKernels[delta->cfg.conv_width - kMinConv], dim3(a.pieces * tiles), dim3(threads), 0,
                       as_stream(stream), a);
    return check_launch("delta_conv");
}

extern "C" tsg_status tsg_delta_decode(tsg_delta* delta, tsg_stream stream,
                                       const tsg_delta_states* states,
                                       const tsg_delta_batch* batch, const tsg_delta_rows* rows,
                                       const float* a_log, const float* dt_bias, uint16_t* out,
                                       uint32_t out_stride) {
    DeltaArgs a{};
    if (tsg_status s = delta_args(delta, states, batch, rows, a_log, dt_bias, out, out_stride, &a))
        return s;
    TSG_REQUIRE(!batch->row_starts, TSG_ERR_INVALID_ARGUMENT,
                "decode takes the same 1...%u rows of every sequence (no row starts)",
                kMaxDeltaKept);
    TSG_REQUIRE(a.seqs.seq_rows <= kMaxDeltaKept, TSG_ERR_DECLINED,
                "more than %u rows a sequence: tsg_delta_prefill", kMaxDeltaKept);
    DeviceScope scope(delta->device);
    TSG_HIP_TRY(scope.status);
    return launch_recurrent(delta, a, stream);
}

extern "C" size_t tsg_delta_prefill_scratch_bytes(const tsg_delta* delta, uint32_t rows,
                                                  uint32_t num_seqs) {
    return delta && rows && num_seqs ? delta_scratch_bytes(delta, rows, num_seqs) : 0u;
}

extern "C" tsg_status tsg_delta_prefill(tsg_delta* delta, tsg_stream stream,
                                        const tsg_delta_states* states,
                                        const tsg_delta_batch* batch, const tsg_delta_rows* rows,
                                        const float* a_log, const float* dt_bias, uint16_t* out,
                                        uint32_t out_stride, void* scratch, size_t scratch_bytes) {
    DeltaArgs a{};
    if (tsg_status s = delta_args(delta, states, batch, rows, a_log, dt_bias, out, out_stride, &a))
        return s;
    TSG_REQUIRE(batch->kept == 1u, TSG_ERR_INVALID_ARGUMENT, "prefill keeps one state a sequence");
    TSG_REQUIRE(scratch && scratch_bytes >=
                               tsg_delta_prefill_scratch_bytes(delta, batch->rows, batch->num_seqs),
                TSG_ERR_INVALID_ARGUMENT, "the scratch is too small");
    TSG_REQUIRE((reinterpret_cast<uintptr_t>(scratch) & 255u) == 0, TSG_ERR_ALIGNMENT,
                "the scratch must be 256-byte aligned");
    DeviceScope scope(delta->device);
    TSG_HIP_TRY(scope.status);
    return launch_chunked(delta, a, scratch, stream);
}

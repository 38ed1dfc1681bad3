// delta_prefill.hip — the gated delta rule over a prompt's rows, 64 at a time.
//
// With G the decays' exponents summed from the chunk's first row, of its rows
//   A_ij = beta_i e^(Gi - Gj) k^i.k^j (j < i),   T = (1 + A)^-1,
//   U = T (beta (V - e^G K^ S)),
//   O = e^G Q^ S + (e^(Gi - Gj) q^i.k^j)_(j <= i) U,   S <- e^(G_end) S + (e^(G_end - G) K^)^T U.
// What does not need the state (T, the weights of O, the rows' factors, K^T in the
// order of the matrix unit) a first kernel forms for all chunks at once into the
// scratch; a second takes the state from chunk to chunk.
//
// The state and what goes into it keep fp32's precision: q and k are fp16 as they are
// (their norms are factors of rows), every other operand is split into two halves of
// fp16 (22 bits; three products where both are split), T and the weights of O are formed in
// fp32, and all sums are in fp32. fp16's range is no limit: a state's columns, R and U are
// scaled by a power of two from bounds on them. |k^| <= 1, beta <= 1 and decays <= 1, so
// a row does not lengthen a column of the state beyond |v|: columns, R and U stay
// within B = sqrt(key_dim) max|S| + 65 max|v|, scaled to 2^13 ... 2^14. |T| and the weights
// are at most 1. Lower halves are kept times 2^11, in the upper ones' range, so that fp16's
// least step leaves out no more than 2^-49 B of an element: B is a column's and a
// chunk's, and rows of one may differ by all of fp16's range (unscaled, the halves end at
// 2^-38 B: one value of 60,000 took all bits from the rows of 1e-3 before it).
#include "delta_internal.hpp"

#include <type_traits>

namespace tsg {
namespace {

constexpr uint32_t kChunk = 64;
// T and the weights are kept times these, away from fp16's least.
constexpr float kTriangle = 32.0f, kWeight = 1024.0f;
// The lower halves of split operands, to the upper ones.
constexpr float kLower = 1.0f / 2048.0f;

// A chunk and value head's record: T's operand pieces and the weights' (two planes each), 64
// lanes x 16 bytes a piece; the rows' factors; e^G_end and how many rows count.
// Pieces (16 rows, 32 columns) of the lower triangle: row tiles 0 and 1 need the first
// column half, 2 and 3 both.
constexpr uint32_t kPieces = 6, kPieceBytes = 1024;
constexpr uint32_t kWeightsAt = 2u * kPieces * kPieceBytes;
constexpr uint32_t kFactorsAt = kWeightsAt + 2u * kPieces * kPieceBytes;
constexpr uint32_t kEndAt = kFactorsAt + 4u * kChunk * 4u;
constexpr uint32_t kRecord = kEndAt + 256u;
__device__ __forceinline__ uint32_t piece_of(uint32_t mt, uint32_t half) {
    return mt < 2u ? mt : 2u * mt - 2u + half;
}
// Pieces of a chunk and key head: K^T's, then K's and Q's (16 rows, 32 elements). In this
// order a wave's load is 1 KiB in a row; the rows as they lie, in 32-byte parts, took the
// address unit three times as long as all else together (8192 rows x 32 heads: 405 us for 260).
template <uint32_t DKP>
constexpr uint32_t kRowsAt = DKP / 16u * 2u * kPieceBytes;
template <uint32_t DKP>
constexpr uint32_t kKeyRecord = kRowsAt<DKP> + 2u * 4u * (DKP / 32u) * kPieceBytes;

struct ChunkArgs {
    DeltaArgs d;
    uint8_t* records;  // [chunk][value head]
    uint8_t* keys;     // [chunk][key head]
    uint32_t key_heads;
    uint32_t chunks;
    uint32_t slices;   // of the value elements, a head
    uint32_t spread;   // heads' workgroups in order, not an XCD each
};

// Lane (i, g)'s eight elements of the matrix unit's operands, i = lane % 16, g = lane
// / 16. Where an accumulator becomes the second operand of the next product, its
// register e of the first and second 16 rows are rows 4 g + e and 16 + 4 g + e of 32:
// the first operand takes its columns in the same order.
__device__ __forceinline__ f4_t mfma(h8_t a, h8_t b, f4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ h8_t as_h8(uint4 u) { return __builtin_bit_cast(h8_t, u); }

// x = hi + kLower lo to 22 bits, or 2^-36. The empty asm keeps the product that x came from
// out of the conversion: rounded once from the exact product in one use and twice in the other,
// the two hi would differ near ties, and lo be what is missing to another hi.
__device__ __forceinline__ void split4(f4_t x, h4_t& hi, h4_t& lo) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float y = x[e];
        asm("" : "+v"(y));
        hi[e] = (_Float16)y;
        lo[e] = (_Float16)(__builtin_fmaf((float)hi[e], -1.0f, y) * (1.0f / kLower));  // exact but for the cast
    }
}

// ------------------------------------------------------- what needs no state

constexpr uint32_t kLd = 68;  // floats of a row of A and T in LDS

// Keys, and in their place the weights, then T; A; what is one a row: four workgroups a CU.
template <uint32_t DKP>
constexpr uint32_t kKeysBytes = std::max(kChunk * (DKP + 8u) * 2u, kChunk * kLd * 4u);
template <uint32_t DKP>
constexpr uint32_t prepare_lds_bytes() {
    return kKeysBytes<DKP> + kChunk * kLd * 4u + 8u * kChunk * 4u + 16u;
}

// x and that of the lane that the DPP control names (0 where there is none).
template <int CTRL, int ROWS>
__device__ __forceinline__ double add_dpp(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, false);
    const uint32_t hi =
        (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, false);
    return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// The sum of the lanes up to this one: from 1, 2, 4 and 8 lanes before within 16, then from
// the last lane of the 16 and of the 32 before.
__device__ __forceinline__ double wave_scan(double x) {
    x = add_dpp<0x111, 0xF>(x);
    x = add_dpp<0x112, 0xF>(x);
    x = add_dpp<0x114, 0xF>(x);
    x = add_dpp<0x118, 0xF>(x);
    x = add_dpp<0x142, 0xA>(x);
    return add_dpp<0x143, 0xC>(x);
}

// A workgroup takes a chunk of a value head; those of one key head, which read the same rows,
// come one after another on one XCD. 8192 rows x 32 heads of 128 x 128: 85 us. Bound by the chain
// of its steps, with four workgroups a CU: the vector units are busy 45 % of the time, LDS 19, the
// matrix units 8 (a key head's value heads in one workgroup, the rows' products once: 220
// registers, 130 us for what then took 91).
template <uint32_t DKP>
__global__ __launch_bounds__(256, 4) void prepare_kernel(ChunkArgs p) {
    constexpr uint32_t KS = DKP + 8u;  // halves of a key row in LDS
    constexpr uint32_t NK = DKP / 32u;
    extern __shared__ __align__(16) uint8_t smem[];
    uint16_t* keys = reinterpret_cast<uint16_t*>(smem);
    float* tm = reinterpret_cast<float*>(smem);
    float* am = reinterpret_cast<float*>(smem + kKeysBytes<DKP>);
    float* wm = tm;  // the weights
    float* k_inv = am + kChunk * kLd;  // 1 / |k|, 1 / |q|
    float *q_inv = k_inv + kChunk, *gs = q_inv + kChunk, *bs = gs + kChunk;
    // of the rows that count for the head (0 for others): no NaN goes into the triangles
    float *g_hi = bs + kChunk, *g_lo = g_hi + kChunk, *rk = g_lo + kChunk, *rq = rk + kChunk;
    uint32_t* valid_at = reinterpret_cast<uint32_t*>(rq + kChunk);  // the head's, the keys'

    const DeltaArgs& d = p.d;
    const uint32_t j8 = blockIdx.x >> 3, unit = j8 / d.group * 8u + (blockIdx.x & 7u);
    const uint32_t chunk = unit / p.key_heads, kh = unit % p.key_heads;
    const uint32_t head = kh * d.group + j8 % d.group;
    if (chunk >= p.chunks) return;
    const DeltaTile t = delta_tile<kChunk>(d.seqs, chunk);
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t i16 = lane & 15u, g = lane >> 4;
    if (t.kind == 2u) {
        if (chunk == 0u && head == 0u && tid == 0u) report(d.seqs.error, kErrDeltaRows);
        const uint32_t pieces = d.value_dim / 8u;
        for (uint32_t n = tid; n < t.count * pieces; n += 256u)
            *reinterpret_cast<uint4*>(d.out + (uint64_t)(t.first + n / pieces) * d.out_stride +
                                      head * d.value_dim + n % pieces * 8u) =
                make_uint4(kDeltaNan2, kDeltaNan2, kDeltaNan2, kDeltaNan2);
        return;
    }
    if (t.count == 0u) return;
    uint8_t* record = p.records + ((uint64_t)chunk * d.value_heads + head) * kRecord;

    // rows: four threads each; norms, gates, keys to LDS
    const uint32_t r = tid >> 2, part = tid & 3u;
    const uint32_t row = t.first + (r < t.count ? r : t.count - 1u);
    if (tid == 0u) valid_at[0] = valid_at[1] = t.count;
    __syncthreads();
    {
        const uint16_t* k = d.k + (uint64_t)row * d.k_stride + kh * d.key_dim;
        const uint16_t* q = d.q + (uint64_t)row * d.q_stride + kh * d.key_dim;
        const uint16_t a_bits = d.a[(uint64_t)row * d.a_stride + head];
        const uint16_t b_bits = d.b[(uint64_t)row * d.b_stride + head];
        float kk = 0.0f, qq = 0.0f;
        uint32_t wrong = 0;
#pragma unroll
        for (uint32_t n = 0; n < DKP / 32u; ++n) {
            const uint32_t c = 8u * (part + 4u * n);
            uint4 u = make_uint4(0, 0, 0, 0), w = u;
            if (c < d.key_dim) {
                u = *reinterpret_cast<const uint4*>(k + c);
                w = *reinterpret_cast<const uint4*>(q + c);
            }
            if (r >= t.count) u = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(keys + r * KS + c) = u;
            const uint32_t us[4] = {u.x, u.y, u.z, u.w}, ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                wrong |= not_finite<false>(us[e]);
                const h2_t x = __builtin_bit_cast(h2_t, us[e]), y = __builtin_bit_cast(h2_t, ws[e]);
                kk = __builtin_fmaf((float)x[0], (float)x[0], kk);
                kk = __builtin_fmaf((float)x[1], (float)x[1], kk);
                qq = __builtin_fmaf((float)y[0], (float)y[0], qq);
                qq = __builtin_fmaf((float)y[1], (float)y[1], qq);
            }
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            kk += __shfl_xor(kk, o, 64);
            qq += __shfl_xor(qq, o, 64);
            wrong |= (uint32_t)__shfl_xor((int)wrong, o, 64);
        }
        if (part == 0u) {
            const float av = f16_to_f32(a_bits) + d.dt_bias[head];
            const float soft = fmaxf(av, 0.0f) + log1pf(expf(-fabsf(av)));
            const float x = av != av ? av : -expf(d.a_log[head]) * 1.44269504f * soft;
            const float beta = 1.0f / (1.0f + expf(-f16_to_f32(b_bits)));
            if ((x != x || beta != beta) && r < t.count) atomicMin(valid_at, r);
            if (wrong) atomicMin(valid_at + 1, r);
            gs[r] = x < -1500.0f ? -1500.0f : x;  // a decay of 2^-1500 is 0
            bs[r] = beta;
            k_inv[r] = 1.0f / sqrtf(kk + d.eps);
            q_inv[r] = 1.0f / sqrtf(qq + d.eps);
        }
    }
    __syncthreads();
    // The head's rows count up to its first wrong gate or key; those behind a wrong key for
    // none of the key head's, so the keys become zeros there.
    const uint32_t key_valid = valid_at[1], valid = key_valid < valid_at[0] ? key_valid : valid_at[0];
    if (key_valid < t.count) {
        if (r >= key_valid)
            for (uint32_t n = 0; n < DKP / 32u; ++n)
                *reinterpret_cast<uint4*>(keys + r * KS + 8u * (part + 4u * n)) = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }

    if (wave == 0u) {
        const bool in = lane < valid;
        // in 64 bits: their differences are what counts
        const double sum = wave_scan(in ? (double)gs[lane] : 0.0);
        const double end = __shfl(sum, 63, 64);
        g_hi[lane] = (float)sum;
        g_lo[lane] = (float)(sum - (double)(float)sum);
        float* f = reinterpret_cast<float*>(record + kFactorsAt) + lane;
        const float since = exp2f((float)sum), until = exp2f((float)(end - sum));
        const float beta = bs[lane], k1 = k_inv[lane];
        // K^T is kept with norms of 2 ... 4, so that U times this stays in fp16's range, and
        // neither's elements near its least
        const int e = __builtin_amdgcn_frexp_expf(1.0f / k1);
        f[0] = in ? beta : 0.0f;
        f[64] = in ? beta * since * k1 : 0.0f;
        f[128] = in ? since * q_inv[lane] * d.scale : 0.0f;
        f[192] = in ? until * __builtin_amdgcn_ldexpf(k1, e - 2) : 0.0f;
        rk[lane] = in ? k1 : 0.0f;
        rq[lane] = in ? q_inv[lane] * kWeight : 0.0f;
        bs[lane] = in ? beta * k1 : 0.0f;
        if (lane == 0u) {
            float* last = reinterpret_cast<float*>(record + kEndAt);
            last[0] = exp2f((float)end);
            last[1] = __uint_as_float(valid);
        }
    }

    // products of the rows' 16-row tiles: K K^T and Q K^T on and below the diagonal
    f4_t kk[4], qk[4];
    const uint32_t mine = 16u * wave + i16, r0 = 16u * wave + 4u * g;
    const uint16_t* q = d.q + (uint64_t)(t.first + (mine < t.count ? mine : t.count - 1u)) * d.q_stride +
                        kh * d.key_dim;
    {
#pragma unroll
        for (uint32_t n = 0; n < 4u; ++n) kk[n] = qk[n] = f4_t{0, 0, 0, 0};
#pragma unroll
        for (uint32_t st = 0; st < NK; ++st) {
            const uint32_t c = 32u * st + 8u * g;
            uint4 qu = make_uint4(0, 0, 0, 0);
            if (c < d.key_dim) qu = *reinterpret_cast<const uint4*>(q + c);
            const h8_t ka = *reinterpret_cast<const h8_t*>(keys + mine * KS + c), qa = as_h8(qu);
#pragma unroll
            for (uint32_t n = 0; n < 4u; ++n) {
                if (n > wave) continue;
                const h8_t kb = *reinterpret_cast<const h8_t*>(keys + (16u * n + i16) * KS + c);
                kk[n] = mfma(ka, kb, kk[n]);
                qk[n] = mfma(qa, kb, qk[n]);
            }
        }
    }
    if (head % d.group == 0u) {
        uint8_t* to = p.keys + ((uint64_t)chunk * p.key_heads + kh) * kKeyRecord<DKP> + lane * 16u;
        for (uint32_t n = wave; n < DKP / 8u; n += 4u) {
            const uint32_t c = 16u * (n / 2u) + i16;
            h8_t x;
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) {
                const uint32_t at = 32u * (n % 2u) + 16u * (e / 4u) + 4u * g + e % 4u;
                const int ex = __builtin_amdgcn_frexp_expf(1.0f / k_inv[at]);
                x[e] = (_Float16)__builtin_amdgcn_ldexpf(f16_to_f32(keys[at * KS + c]), 2 - ex);
            }
            *reinterpret_cast<h8_t*>(to + n * kPieceBytes) = x;
        }
        to += kRowsAt<DKP>;
#pragma unroll
        for (uint32_t st = 0; st < NK; ++st) {
            uint2 a[4];
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h) {
                const uint32_t c = 32u * st + 16u * h + 4u * g;
                a[h] = *reinterpret_cast<const uint2*>(keys + mine * KS + c);
                a[2u + h] = make_uint2(0, 0);
                if (c < d.key_dim) a[2u + h] = *reinterpret_cast<const uint2*>(q + c);
            }
            uint8_t* at = to + (wave * NK + st) * kPieceBytes;
            *reinterpret_cast<uint4*>(at) = make_uint4(a[0].x, a[0].y, a[1].x, a[1].y);
            *reinterpret_cast<uint4*>(at + 4u * NK * kPieceBytes) =
                make_uint4(a[2].x, a[2].y, a[3].x, a[3].y);
        }
    }

    __syncthreads();
    {
        const f4_t hi = *reinterpret_cast<const f4_t*>(g_hi + r0);
        const f4_t lo = *reinterpret_cast<const f4_t*>(g_lo + r0);
        const f4_t bi = *reinterpret_cast<const f4_t*>(bs + r0);
        const f4_t qi = *reinterpret_cast<const f4_t*>(rq + r0);
        float hj[4], lj[4], kj[4];
#pragma unroll
        for (uint32_t n = 0; n < 4u; ++n) {
            hj[n] = g_hi[16u * n + i16];
            lj[n] = g_lo[16u * n + i16];
            kj[n] = rk[16u * n + i16];
        }
#pragma unroll
        for (uint32_t n = 0; n < 4u; ++n) {
            const uint32_t j = 16u * n + i16;
            if (n > wave) {
                if ((n ^ 1u) != wave) continue;  // the other half of a piece
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e) wm[(r0 + e) * kLd + j] = 0.0f;
                continue;
            }
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e) {
                const uint32_t i = r0 + e;
                const float w =
                    __builtin_amdgcn_exp2f(i >= j ? (hi[e] - hj[n]) + (lo[e] - lj[n]) : 0.0f) * kj[n];
                am[i * kLd + j] = i > j ? bi[e] * w * kk[n][e] : 0.0f;
                // a query's infinity or NaN stays in its row's weights
                wm[i * kLd + j] = i >= j ? qi[e] * w * qk[n][e] : 0.0f;
            }
        }
    }
    __syncthreads();
    // A triangle's pieces, in two planes.
    const auto put_pieces = [&](const float* m, float times, uint8_t* to) {
        for (uint32_t n = wave; n < kPieces; n += 4u) {
            const uint32_t mt = n < 2u ? n : 2u + (n - 2u) / 2u, half = n < 2u ? 0u : n % 2u;
            const float* src = m + (16u * mt + i16) * kLd + 32u * half + 4u * g;
            h4_t hi[2], lo[2];
#pragma unroll
            for (uint32_t e = 0; e < 2u; ++e)
                split4(*reinterpret_cast<const f4_t*>(src + 16u * e) * times, hi[e], lo[e]);
            h4_t* o = reinterpret_cast<h4_t*>(to + n * kPieceBytes + lane * 16u);
            o[0] = hi[0];
            o[1] = hi[1];
            o += kPieces * kPieceBytes / 8u;
            o[0] = lo[0];
            o[1] = lo[1];
        }
    };
    put_pieces(wm, 1.0f, record + kWeightsAt);

    __syncthreads();  // T takes the weights' place
    // T: the diagonal tiles by substitution, a column a lane, ...
    {
        float x[16];
#pragma unroll
        for (uint32_t i = 0; i < 16u; ++i) {
            float y = i == i16 ? 1.0f : 0.0f;
            const float* a = am + (16u * wave + i) * kLd + 16u * wave;
#pragma unroll
            for (uint32_t j = 0; j < i; ++j) y = __builtin_fmaf(-a[j], x[j], y);
            x[i] = y;
        }
#pragma unroll
        for (uint32_t i = 0; i < 16u; ++i)
            if (i / 4u == g) tm[(16u * wave + i) * kLd + 16u * wave + i16] = x[i];
        if (wave == 0u || wave == 2u) {  // beside them zeros, the other half of a piece
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e)
                tm[(16u * wave + 4u * g + e) * kLd + 16u * wave + 16u + i16] = 0.0f;
        }
    }
    __syncthreads();
    // ... then T_21 = -T_22 A_21 T_11, of tiles of 16 and of 32. Tile products in fp32.
    const auto first4 = [&](const float* m, uint32_t mt, uint32_t kt) {
        return *reinterpret_cast<const f4_t*>(m + (16u * mt + i16) * kLd + 16u * kt + 4u * g);
    };
    const auto from_lds = [&](f4_t c, const float* a, uint32_t mt, uint32_t kt, const float* b,
                              uint32_t nt) {
        const f4_t x = first4(a, mt, kt);
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(
                x[e], b[(16u * kt + 4u * g + e) * kLd + 16u * nt + i16], c, 0, 0, 0);
        return c;
    };
    const auto from_regs = [&](f4_t c, const float* a, uint32_t mt, uint32_t kt, f4_t b) {
        const f4_t x = first4(a, mt, kt);
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], b[e], c, 0, 0, 0);
        return c;
    };
    const auto put = [&](f4_t y, uint32_t mt, uint32_t nt) {
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) tm[(16u * mt + 4u * g + e) * kLd + 16u * nt + i16] = -y[e];
    };
    const f4_t none = f4_t{0, 0, 0, 0};
    if (wave < 2u) {
        const uint32_t b = 2u * wave;
        put(from_regs(none, tm, b + 1u, b + 1u, from_lds(none, am, b + 1u, b, tm, b)), b + 1u, b);
    }
    __syncthreads();
    {
        const uint32_t mt = 2u + (wave >> 1), nt = wave & 1u;
        f4_t x2 = from_lds(none, am, 2u, 1u, tm, nt), x3 = from_lds(none, am, 3u, 1u, tm, nt);
        if (nt == 0u) {
            x2 = from_lds(x2, am, 2u, 0u, tm, 0u);
            x3 = from_lds(x3, am, 3u, 0u, tm, 0u);
        }
        f4_t y = from_regs(none, tm, mt, 2u, x2);
        if (mt == 3u) y = from_regs(y, tm, 3u, 3u, x3);
        put(y, mt, nt);
    }
    __syncthreads();
    put_pieces(tm, kTriangle, record);
}

// ------------------------------------------------------- from chunk to chunk
//
// A workgroup takes 16 value elements of a sequence and head. Each of its eight waves
// holds an eighth of the state's key rows in registers and multiplies 16 rows of K (waves 0
// to 3) or of Q with the state; the first four go on to U, the others to the outputs. What
// one wave's products need of the others' goes through LDS as operands of the matrix unit,
// three exchanges a chunk: S, then R = beta (V - e^G K^ S), then U. Operands of the next
// chunk are loaded as soon as this one's are used. 8192 rows x 32 heads of 128 x 128: 214 us, 1.7
// a chunk with one workgroup a CU; 7 prompts of 11207 rows 271, 1.5 with two. Bound by the
// operands' way from L2, 84 KB a chunk and workgroup, 12 and 14 TB/s in these two: the
// outputs' weights in two halves, 7 % more of them, took 8 % more time, where the chains of
// products and the place of the outputs' step changed nothing. Vector units are busy 40 and 51 % of
// the time, LDS 30 and 36 (conflicts 7 and 8), matrix units 13 and 16. When a chunk took 75 KB:
// four waves for both roles 260 us for 202; 32 columns a workgroup, which halve the loads, but
// of which one fits a CU, 292 for 268 (the prompts).

constexpr uint32_t kScanThreads = 512;

// The sequence of the n-th most rows, of up to 64: the longest chains are begun first (7
// prompts of 201 to 3001 rows 251 us, in order 262, at 75 KB of operands a chunk).
__device__ __forceinline__ uint32_t longest_first(const DeltaSeqs& d, uint32_t n) {
    const uint32_t lane = threadIdx.x & 63u;
    const bool live = lane < d.num_seqs;
    const uint32_t count = live ? d.row_starts[lane + 1u] - d.row_starts[lane] : 0u;
    uint32_t rank = 0;
    for (uint32_t j = 0; j < d.num_seqs; ++j) {
        const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)count, (int)j);
        rank += other > count || (other == count && j < lane) ? 1u : 0u;
    }
    return (uint32_t)__builtin_ctzll(__ballot(live && rank == n));
}

template <uint32_t DKP>
__global__ __launch_bounds__(kScanThreads, (DKP <= 128u ? 4 : 2)) void scan_kernel(ChunkArgs p) {
    constexpr uint32_t NK = DKP / 32u;                 // key steps
    constexpr uint32_t TW = DKP <= 128u ? 1u : 2u;     // state tiles (16 key rows) of a wave
    constexpr uint32_t SHARE = 2u * kPieceBytes;       // two planes of a piece
    __shared__ __align__(16) uint8_t s_at[NK * SHARE];
    __shared__ __align__(16) uint8_t r_at[2u * SHARE];
    __shared__ __align__(16) uint8_t u_at[2][2u * SHARE];  // U, for the outputs, of two chunks
    __shared__ __align__(16) uint8_t w_at[2u * SHARE];  // U times the rows' factors, for the state
    __shared__ __align__(16) float most[16][8];         // [column]: |S| of the waves
    __shared__ __align__(16) float v_most_at[2][16][4];  // |v| of the row tiles, of two chunks
    __shared__ float rare[16][8];
    __shared__ __align__(16) float factors[4][kChunk];  // of V, K S, Q S and U, a chunk's
    // 16 rows and columns of V and O, between a lane's place in memory (four elements of
    // row lane / 4) and in the matrix unit: one access of 8 bytes a lane for four of 2.
    __shared__ __align__(16) uint16_t v_at[2][4][16][20];  // [column][row], of two chunks
    __shared__ __align__(16) uint16_t o_at[4][16][20];  // [row][column]

    const DeltaArgs& d = p.d;
    const uint32_t lane = threadIdx.x & 63u, i16 = lane & 15u, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t rt = wave & 3u;                 // the wave's tile of 16 rows
    const bool holds = DKP >= 128u || wave < 4u;   // a part of the state
    // Workgroups go to the XCDs in turn: those of one key head share its rows there.
    const uint32_t inner = d.group * p.slices;
    uint32_t unit = blockIdx.x / inner, at = blockIdx.x % inner;
    if (!p.spread) {
        const uint32_t j = blockIdx.x >> 3;
        unit = j / inner * 8u + (blockIdx.x & 7u);
        at = j % inner;
    }
    uint32_t s = unit / p.key_heads;
    const uint32_t kh = unit % p.key_heads;
    if (s >= d.seqs.num_seqs) return;
    const uint32_t head = kh * d.group + at / p.slices, c0 = at % p.slices * 16u;
    if (starts_wrong(d.seqs)) return;  // reported, and the rows made NaN, by the first kernel
    if (d.seqs.row_starts && d.seqs.num_seqs <= 64u) s = longest_first(d.seqs, s);
    const DeltaSeq sq = delta_seq(d.seqs, s);
    const bool bad = out_slots_clash<1u>(d.seqs, s) || sq.bad;
    const uint32_t col4 = head * d.value_dim + c0 + 4u * (lane & 3u);
    if (bad) {
        if (at == 0u && kh == 0u && threadIdx.x == 0u) report(d.seqs.error, kErrDeltaSlot);
        for (uint32_t r = threadIdx.x >> 2; r < sq.count; r += kScanThreads / 4u)
            *reinterpret_cast<uint2*>(d.out + (uint64_t)(sq.first + r) * d.out_stride + col4) =
                make_uint2(kDeltaNan2, kDeltaNan2);
        return;
    }

    // the state: register e of tile t of the wave's is key row 16 (TW wave + t) + 4 g + e, times
    // 2^(14 - exponent), the exponent of the column's last bound
    const uint64_t place = (uint64_t)head * d.key_dim * d.value_dim + c0 + i16;
    if (sq.count == 0u) {  // handed on as it is
        const uint32_t slot = scalar_load(d.seqs.out_slots + s);
        if (slot == TSG_NO_SLOT) return;
        for (uint32_t kr = threadIdx.x >> 4; kr < d.key_dim; kr += kScanThreads / 16u) {
            const uint64_t at_kr = place + kr * d.value_dim;
            d.s[(uint64_t)slot * d.slot_stride + at_kr] =
                sq.fresh ? 0.0f : d.s[(uint64_t)sq.in * d.slot_stride + at_kr];
        }
        return;
    }
    f4_t st[TW];
    const auto column_most = [&] {
        float m = 0.0f;
#pragma unroll
        for (uint32_t t = 0; t < TW; ++t)
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e) m = fmaxf(m, fabsf(st[t][e]));
        return max_across32(max_across16(m));
    };

    const uint32_t chunks = (sq.count + kChunk - 1u) / kChunk;
    const uint32_t chunk0 = delta_tile_base<kChunk>(d.seqs, sq, s);
    // Loads: a place that is the same for the wave, and the lane's within it.
    const uint32_t lane16 = lane * 16u;
    const auto piece = [](const uint8_t* base, uint32_t off) {
        return *reinterpret_cast<const h8_t*>(base + off);
    };
    const auto record = [&](uint32_t c) {
        return p.records + ((uint64_t)(chunk0 + c) * d.value_heads + head) * kRecord;
    };
    const auto key_record = [&](uint32_t c) {
        return p.keys + ((uint64_t)(chunk0 + c) * p.key_heads + kh) * kKeyRecord<DKP>;
    };
    // a split value's planes as the second operand: the wave's tile of 16 rows
    const auto share = [&](uint8_t* to, uint32_t tile, f4_t x) {
        h4_t hi, lo;
        split4(x, hi, lo);
        uint8_t* o = to + tile / 2u * SHARE + tile % 2u * 8u + lane16;
        *reinterpret_cast<h4_t*>(o) = hi;
        *reinterpret_cast<h4_t*>(o + kPieceBytes) = lo;
    };
    const auto shared_piece = [&](const uint8_t* from, uint32_t step, uint32_t plane) {
        return *reinterpret_cast<const h8_t*>(from + step * SHARE + plane * kPieceBytes + lane16);
    };

    const float reach = sqrtf((float)d.key_dim) * 1.01f;
#pragma unroll
    for (uint32_t t = 0; t < TW; ++t)
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) {
            const uint32_t kr = 16u * (TW * wave + t) + 4u * g + e;
            st[t][e] = !sq.fresh && kr < d.key_dim
                           ? d.s[(uint64_t)sq.in * d.slot_stride + place + kr * d.value_dim]
                           : 0.0f;
        }
    const auto most_of_waves = [&] {
        const f4_t a = *reinterpret_cast<const f4_t*>(&most[i16][0]);
        const f4_t b = *reinterpret_cast<const f4_t*>(&most[i16][4]);
        return fmaxf(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])),
                     fmaxf(fmaxf(b[0], b[1]), fmaxf(b[2], b[3])));
    };
    const float m_first = column_most();
    if (g == 0u) most[i16][wave] = m_first;
    lds_barrier();
    int exponent = __builtin_amdgcn_frexp_expf(most_of_waves());
    exponent = exponent > -100 ? exponent : -100;
    lds_barrier();
#pragma unroll
    for (uint32_t t = 0; t < TW; ++t) st[t] *= __builtin_amdgcn_ldexpf(1.0f, 14 - exponent);

    // The loop, of the waves of keys and of queries: each its own code, so that a wait counts
    // the loads of its own only, with the same barriers.
    const auto run = [&](auto role) {
        constexpr bool keys = decltype(role)::value;
        const bool two = rt >= 2u;  // the wave's rows see both halves of the chunk's
        h8_t rf[NK], th[2], tl[2], kt[TW][2];  // rows of K or Q; T or the weights; K^T
        uint2 v_row = make_uint2(0, 0);
        float f_row = 0.0f;
        const uint32_t rows_at = kRowsAt<DKP> + wave * NK * kPieceBytes;
        const auto load_rows = [&](uint32_t c) {
            const uint8_t* k = key_record(c) + rows_at;
#pragma unroll
            for (uint32_t n = 0; n < NK; ++n) rf[n] = piece(k + n * kPieceBytes, lane16);
        };
        // the waves of queries also bring the values and the rows' factors
        const auto load_v = [&](uint32_t c) {
            if constexpr (!keys) {
                const uint32_t base = kChunk * c + 16u * rt;
                const uint32_t left = sq.count > base ? sq.count - base : 0u;
                const uint32_t first = left ? base : sq.count - 1u;  // the last row in the place of none
                uint32_t r = lane >> 2;
                r = r < left ? r : left ? left - 1u : 0u;
                v_row = *reinterpret_cast<const uint2*>(
                    reinterpret_cast<const uint8_t*>(d.v + (uint64_t)(sq.first + first) * d.v_stride) +
                    2u * (r * d.v_stride + col4));
            }
        };
        const auto load_factors = [&](uint32_t c) {
            if constexpr (!keys)
                f_row = *reinterpret_cast<const float*>(record(c) + kFactorsAt + 256u * rt + 4u * lane);
        };
        // the loaded values' columns, and the largest of each
        const auto turn_v = [&](uint32_t c) {
            uint16_t(*v)[20] = v_at[c & 1u][rt];
            const uint32_t r = lane >> 2, c4 = 4u * (lane & 3u);
            v[c4][r] = (uint16_t)v_row.x;
            v[c4 + 1u][r] = (uint16_t)(v_row.x >> 16);
            v[c4 + 2u][r] = (uint16_t)v_row.y;
            v[c4 + 3u][r] = (uint16_t)(v_row.y >> 16);
            __builtin_amdgcn_wave_barrier();
            const uint2 u = *reinterpret_cast<const uint2*>(&v[i16][4u * g]);
            const uint32_t b[4] = {u.x & 0x7FFFu, u.x >> 16 & 0x7FFFu, u.y & 0x7FFFu, u.y >> 16 & 0x7FFFu};
            uint32_t bits = 0;
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e) bits = bits > b[e] ? bits : b[e];
            // infinities and NaN count as infinity
            const float mv = max_across32(max_across16(
                bits < 0x7C00u ? f16_to_f32((uint16_t)bits) : __builtin_inff()));
            if (g == 0u) v_most_at[c & 1u][i16][rt] = mv;
        };
        const uint32_t t_0 = piece_of(rt, 0u) * kPieceBytes, t_1 = piece_of(rt, two ? 1u : 0u) * kPieceBytes;
        const auto load_t = [&](uint32_t c) {
            const uint8_t* r = record(c) + (keys ? 0u : kWeightsAt);
            th[0] = piece(r + t_0, lane16);
            tl[0] = piece(r + t_0 + kPieces * kPieceBytes, lane16);
            th[1] = piece(r + t_1, lane16);
            tl[1] = piece(r + t_1 + kPieces * kPieceBytes, lane16);
        };
        const auto load_k = [&](uint32_t c) {
            const uint8_t* k = key_record(c) + (holds ? TW * wave * SHARE : 0u);
#pragma unroll
            for (uint32_t t = 0; t < TW; ++t)
#pragma unroll
                for (uint32_t h = 0; h < 2u; ++h) kt[t][h] = piece(k + (2u * t + h) * kPieceBytes, lane16);
        };
        // the rows of T or the weights times what is shared: x + kLower x2
        const auto triangle = [&](const uint8_t* from, f4_t& x, f4_t& x2) {
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h) {
                if (h && !two) continue;
                const h8_t hi = shared_piece(from, h, 0u), lo = shared_piece(from, h, 1u);
                x = mfma(th[h], hi, x);
                x2 = mfma(tl[h], hi, x2);
                x2 = mfma(th[h], lo, x2);
            }
        };
        // A chunk's outputs: Q S, and the weights times U, one chunk later while the waves of
        // keys form U.
        f4_t o = {0, 0, 0, 0}, o_next = {0, 0, 0, 0};
        float o_unit = 0.0f;
        uint32_t o_good = 0;
        const auto finish = [&](uint32_t c) {
            f4_t y = {0, 0, 0, 0}, y2 = {0, 0, 0, 0};
            triangle(u_at[c & 1u], y, y2);
            const uint32_t base = kChunk * c + 16u * rt;
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e) {
                o[e] = __builtin_fmaf(__builtin_fmaf(y2[e], kLower, y[e]), o_unit, o[e]);
                if (16u * rt + 4u * g + e >= o_good) o[e] = __builtin_nanf("");
                o_at[rt][4u * g + e][i16] = f32_to_f16(o[e]);
            }
            __builtin_amdgcn_wave_barrier();
            if (base + (lane >> 2) < sq.count)
                *reinterpret_cast<uint2*>(
                    reinterpret_cast<uint8_t*>(d.out + (uint64_t)(sq.first + base) * d.out_stride) +
                    2u * ((lane >> 2) * d.out_stride + col4)) =
                    *reinterpret_cast<const uint2*>(&o_at[rt][lane >> 2][4u * (lane & 3u)]);
            __builtin_amdgcn_wave_barrier();
        };
        load_v(0u);
        if constexpr (!keys) turn_v(0u);
        load_rows(0u);
        load_factors(0u);
        load_v(chunks > 1u ? 1u : 0u);
        load_t(0u);
        load_k(0u);
#pragma unroll 1
        for (uint32_t c = 0; c < chunks; ++c) {
            const uint32_t next = c + 1u < chunks ? c + 1u : c;
            const uint32_t* last = reinterpret_cast<const uint32_t*>(record(c) + kEndAt);
            const float end_decay = __uint_as_float(scalar_load(last));
            const uint32_t valid = scalar_load(last + 1);
            const uint32_t r0 = 16u * rt + 4u * g;  // the lane's rows of the chunk: r0 .. r0 + 3

            // S, and the sizes of its columns and of the values
            if (holds) {
#pragma unroll
                for (uint32_t t = 0; t < TW; ++t) share(s_at, TW * wave + t, st[t]);
            }
            {
                const float ms = column_most();
                if (g == 0u) most[i16][wave] = ms;
            }
            if constexpr (!keys) factors[rt][lane] = f_row;
            lds_barrier();
            // the rows' products with S: of K or of Q
            f4_t ps = {0, 0, 0, 0}, ps2 = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t n = 0; n < NK; ++n) {
                ps = mfma(rf[n], shared_piece(s_at, n, 0u), ps);
                ps2 = mfma(rf[n], shared_piece(s_at, n, 1u), ps2);
            }
            ps += ps2 * kLower;
            load_rows(next);
            uint2 vs = make_uint2(0, 0);  // the lane's values
            if constexpr (keys) vs = *reinterpret_cast<const uint2*>(&v_at[c & 1u][rt][i16][4u * g]);
            uint32_t vb[4] = {vs.x & 0xFFFFu, vs.x >> 16, vs.y & 0xFFFFu, vs.y >> 16};
            const f4_t mb = *reinterpret_cast<const f4_t*>(&v_most_at[c & 1u][i16][0]);
            float v_most = fmaxf(fmaxf(mb[0], mb[1]), fmaxf(mb[2], mb[3]));
            uint32_t first_bad = kChunk;  // row of the column's first infinity or NaN
            if (__ballot(v_most == __builtin_inff())) {  // the same in all waves
                if constexpr (keys) {
                    uint32_t from = kChunk;
                    float fine = 0.0f;
#pragma unroll
                    for (uint32_t e = 0; e < 4u; ++e) {
                        const uint32_t b = vb[e] & 0x7FFFu;
                        if (b >= 0x7C00u) from = from < r0 + e ? from : r0 + e;
                        else fine = fmaxf(fine, f16_to_f32((uint16_t)b));
                    }
                    fine = max_across32(max_across16(fine));
                    const float first = -max_across32(max_across16(-(float)from));
                    if (g == 0u) {
                        rare[i16][rt] = first;
                        rare[i16][4u + rt] = fine;
                    }
                }
                lds_barrier();
                v_most = 0.0f;
#pragma unroll
                for (uint32_t w = 0; w < 4u; ++w) {
                    const uint32_t b = (uint32_t)rare[i16][w];
                    first_bad = first_bad < b ? first_bad : b;
                    v_most = fmaxf(v_most, rare[i16][4u + w]);
                }
                lds_barrier();
                if constexpr (keys) {
#pragma unroll
                    for (uint32_t e = 0; e < 4u; ++e) vb[e] = r0 + e < first_bad ? vb[e] : 0u;
                }
            }
            const uint32_t good = valid < first_bad ? valid : first_bad;
            // the bound on U and on the next S; no further below the last than fp32 has room for
            const float from_s = __builtin_amdgcn_ldexpf(1.0f, exponent - 14);
            int now = __builtin_amdgcn_frexp_expf(most_of_waves() * (reach * from_s) + 65.0f * v_most);
            now = now > -100 ? now : -100;
            now = now > exponent - 60 ? now : exponent - 60;
            const float ratio = __builtin_amdgcn_ldexpf(1.0f, exponent - now);
            exponent = now;
            if constexpr (keys) {
                const float to_r = __builtin_amdgcn_ldexpf(1.0f, 14 - now);
                const f4_t f_v = *reinterpret_cast<const f4_t*>(&factors[0][r0]) * to_r;
                const f4_t f_s = *reinterpret_cast<const f4_t*>(&factors[1][r0]) * ratio;
                f4_t x;
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e)  // 0 for rows that do not count: their factors are
                    x[e] = __builtin_fmaf(f16_to_f32((uint16_t)vb[e]), f_v[e],
                                          -ps[e] * f_s[e]);
                share(r_at, rt, x);
            } else {
                o_next = ps * (*reinterpret_cast<const f4_t*>(&factors[2][r0]) * from_s);
                turn_v(c + 1u);  // the next chunk's
            }
            load_factors(next);
            load_v(c + 2u < chunks ? c + 2u : next);
            lds_barrier();
            if constexpr (keys) {
                f4_t u = {0, 0, 0, 0}, u2 = {0, 0, 0, 0};
                triangle(r_at, u, u2);
                u = (u + u2 * kLower) * (1.0f / kTriangle);
                share(w_at, rt, u * *reinterpret_cast<const f4_t*>(&factors[3][r0]));
                share(u_at[c & 1u], rt, u);
            } else {
                if (c) finish(c - 1u);
                o = o_next;
                o_unit = d.scale * __builtin_amdgcn_ldexpf(1.0f / kWeight, now - 14);
                o_good = good;
            }
            load_t(keys ? next : c);
            lds_barrier();
            f4_t more[TW], more2[TW];
#pragma unroll
            for (uint32_t t = 0; t < TW; ++t) {
                more[t] = st[t] * (end_decay * ratio);
                more2[t] = f4_t{0, 0, 0, 0};
            }
            if (holds) {
#pragma unroll
                for (uint32_t h = 0; h < 2u; ++h) {
                    const h8_t hi = shared_piece(w_at, h, 0u), lo = shared_piece(w_at, h, 1u);
#pragma unroll
                    for (uint32_t t = 0; t < TW; ++t) {
                        more2[t] = mfma(kt[t][h], lo, more2[t]);
                        more[t] = mfma(kt[t][h], hi, more[t]);
                    }
                }
            }
            load_k(next);
            // rows that do not count for what they hold
            const uint32_t rows = sq.count - kChunk * c;
            const bool lost = good < (rows < kChunk ? rows : kChunk);
#pragma unroll
            for (uint32_t t = 0; t < TW; ++t) st[t] = more[t] + more2[t] * kLower;
            if (__ballot(lost)) {
#pragma unroll
                for (uint32_t t = 0; t < TW; ++t)
#pragma unroll
                    for (uint32_t e = 0; e < 4u; ++e)
                        if (lost) st[t][e] = __builtin_nanf("");
            }
        }
        if constexpr (!keys) finish(chunks - 1u);
    };
    __builtin_amdgcn_s_waitcnt(0x0F70);
    if (wave < 4u) run(std::true_type());
    else run(std::false_type());
    const uint32_t slot = scalar_load(d.seqs.out_slots + s);
    if (slot == TSG_NO_SLOT) return;
    const float from_s = __builtin_amdgcn_ldexpf(1.0f, exponent - 14);
    // the lane anew: kept over the loop, its places take registers that the loop lacks
    const uint32_t now = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    float* to = d.s + (uint64_t)slot * d.slot_stride + (uint64_t)head * d.key_dim * d.value_dim + c0;
#pragma unroll
    for (uint32_t t = 0; t < TW; ++t)
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) {
            const uint32_t kr = 16u * (TW * wave + t) + 4u * (now >> 4) + e;
            if (kr < d.key_dim) to[(now & 15u) + kr * d.value_dim] = st[t][e] * from_s;
        }
}

template <uint32_t DKP>
constexpr uint64_t chunk_bytes(uint64_t value_heads, uint64_t key_heads) {
    return value_heads * kRecord + key_heads * kKeyRecord<DKP>;
}

template <uint32_t DKP>
tsg_status launch(const tsg_delta* delta, ChunkArgs p, uint32_t chunks, tsg_stream stream) {
    p.keys = p.records + (uint64_t)chunks * p.d.value_heads * kRecord;
    const uint64_t prepared = ((uint64_t)chunks * p.key_heads + 7u) / 8u * 8u * p.d.group;
    TSG_REQUIRE(prepared <= kMaxBlocks, TSG_ERR_UNSUPPORTED, "too many rows and heads for one launch");
    const uint64_t units = (uint64_t)p.d.seqs.num_seqs * p.key_heads;
    const uint64_t inner = (uint64_t)p.d.group * p.slices;
    p.spread = units % 8u && units < 64u ? 1u : 0u;
    const uint64_t blocks = p.spread ? units * inner : (units + 7u) / 8u * 8u * inner;
    TSG_REQUIRE(2u * blocks <= kMaxBlocks, TSG_ERR_UNSUPPORTED,
                "too many sequences and heads for one launch");
    p.chunks = chunks;
    hipLaunchKernelGGL(prepare_kernel<DKP>, dim3((uint32_t)prepared), dim3(256),
                       prepare_lds_bytes<DKP>(), as_stream(stream), p);
    if (tsg_status s = check_launch("delta_prepare")) return s;
    hipLaunchKernelGGL(scan_kernel<DKP>, dim3((uint32_t)blocks), dim3(kScanThreads), 0, as_stream(stream), p);
    return check_launch("delta_scan");
}

}  // namespace

uint64_t delta_scratch_bytes(const tsg_delta* delta, uint32_t rows, uint32_t num_seqs) {
    const uint64_t chunks = (uint64_t)rows / kChunk + num_seqs;
    const uint64_t hv = delta->cfg.value_heads, hk = delta->cfg.key_heads;
    return chunks * (delta->padded_key == 64u    ? chunk_bytes<64>(hv, hk)
                     : delta->padded_key == 128u ? chunk_bytes<128>(hv, hk)
                                                 : chunk_bytes<256>(hv, hk));
}

tsg_status prepare_delta(const tsg_delta* delta) {
    const auto kernel = delta->padded_key == 64u    ? prepare_kernel<64>
                        : delta->padded_key == 128u ? prepare_kernel<128>
                                                    : prepare_kernel<256>;
    const uint32_t lds = delta->padded_key == 64u    ? prepare_lds_bytes<64>()
                         : delta->padded_key == 128u ? prepare_lds_bytes<128>()
                                                     : prepare_lds_bytes<256>();
    TSG_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    return TSG_OK;
}

tsg_status launch_chunked(const tsg_delta* delta, const DeltaArgs& a, void* scratch,
                          tsg_stream stream) {
    ChunkArgs p{};
    p.d = a;
    p.records = static_cast<uint8_t*>(scratch);
    p.key_heads = delta->cfg.key_heads;
    p.slices = a.value_dim / 16u;
    const uint32_t chunks = delta_tiles<kChunk>(a.seqs.rows, a.seqs.num_seqs, a.seqs.seq_rows,
                                                a.seqs.row_starts != nullptr);
    switch (delta->padded_key) {
        case 64: return launch<64>(delta, p, chunks, stream);
        case 128: return launch<128>(delta, p, chunks, stream);
        default: return launch<256>(delta, p, chunks, stream);
    }
}

}  // namespace tsg

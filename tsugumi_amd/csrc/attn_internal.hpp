// attn_internal.hpp — what the attention's translation units share: the plan
// object, the kernels' arguments and the device's view of a batch.
#pragma once

#include "tsg_internal.hpp"

struct tsg_attn {
    tsg_ctx* ctx = nullptr;
    int device = 0;  // the context's
    tsg_attn_config cfg{};
    uint32_t group = 0;       // query heads a key head serves
    uint32_t page_shift = 0;  // log2(page_tokens)
    uint32_t cell = 2;        // bytes of a cache element
    uint32_t padded_dim = 64; // the kernels' head width: 64, 128, 256 or 512
    // scratch of the calls that split the keys: partial results and arrival
    // counters (zeroed once, left zeroed by each call)
    float* partials = nullptr;
    uint32_t* arrivals = nullptr;
};

namespace tsg {

// Bits of the context's error word (beside the kErr* of tsg_internal.hpp): a
// page id past the pool or a sequence longer than its page table (its rows
// are NaN, and nothing of them is appended); row starts that fall or pass the
// batch's rows.
constexpr uint32_t kErrAttnPage = 256u;
constexpr uint32_t kErrAttnLength = 512u;
constexpr uint32_t kErrAttnRows = 1024u;

constexpr uint32_t kMaxDecodeRows = 8;  // rows a sequence in a decode call (a speculative block)

struct AttnArgs {
    const uint16_t* q;
    uint16_t* out;
    const uint8_t* k;
    const uint8_t* v;
    const uint32_t* table;
    const uint32_t* lengths;
    const uint32_t* row_starts;  // nullptr: uniform rows a sequence
    uint32_t* error;
    uint64_t page_stride, head_stride;  // bytes
    uint32_t token_stride;              // bytes
    uint32_t q_stride, out_stride;      // elements
    uint32_t table_stride, num_seqs, rows, seq_rows, num_pages;
    uint32_t q_heads, kv_heads, group, dim, page_shift;
    uint32_t window, sinks;
    // q . k to logits in powers of two: |scale| k_scale log2(e), at least 1e-30
    // so that a masked product of -inf stays -inf; a negative scale turns q
    float scale_log2;
    uint32_t q_sign;  // 0x80008000 where the scale is negative
    float v_scale;
};

// A word that no kernel writes meanwhile, at an address that is the same for
// the wave, by a scalar load.
typedef __attribute__((address_space(4))) const uint32_t const_u32_t;
__device__ __forceinline__ uint32_t scalar_load(const uint32_t* p) {
    return *(const_u32_t*)(uintptr_t)p;
}

struct SeqRows {
    uint32_t seq, first, count;  // its rows are first .. first + count - 1
    uint32_t length;             // tokens in the cache
    uint32_t bad;                // kErrAttnLength, kErrAttnRows or 0
};

// Rows and length of sequence s. Every value read from device memory is held
// to the batch's bounds before it is used.
__device__ __forceinline__ SeqRows seq_rows(const uint32_t* row_starts, const uint32_t* lengths,
                                            uint32_t s, uint32_t uniform, uint32_t rows,
                                            uint32_t capacity) {
    SeqRows r;
    r.seq = s;
    r.bad = 0u;
    if (row_starts) {
        const uint32_t lo = scalar_load(row_starts + s), hi = scalar_load(row_starts + s + 1u);
        if (lo > hi || hi > rows) r.bad = kErrAttnRows;
        r.first = lo < rows ? lo : rows;
        const uint32_t end = hi < rows ? hi : rows;
        r.count = end > r.first ? end - r.first : 0u;
    } else {
        r.first = s * uniform;
        r.count = uniform;
    }
    const uint32_t n = scalar_load(lengths + s);
    if (n > capacity) r.bad = kErrAttnLength;
    r.length = n > capacity ? capacity : n;
    return r;
}

__device__ __forceinline__ void report(uint32_t* error, uint32_t bit) { atomicOr(error, bit); }

// The sequence that holds `row` (uniform over the wave), or num_seqs: with row
// starts the last s that starts at or before the row, 64 of them at a time from
// the last. Starts that fall or pass the batch's rows make those before them
// meaningless: a row before the sequences behind the last such one is `broken`.
// The waves of row 0 look at all starts and report.
__device__ __forceinline__ uint32_t find_seq(const uint32_t* row_starts, uint32_t num_seqs,
                                             uint32_t uniform, uint32_t rows, uint32_t row,
                                             uint32_t* error, bool* broken) {
    *broken = false;
    if (!row_starts) return row / uniform;
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t found = num_seqs;
    bool done = false;
    for (uint32_t base = 0; base < num_seqs; base += 64u) {
        const bool live = base + lane < num_seqs;
        const uint32_t s = live ? num_seqs - 1u - (base + lane) : 0u;
        const uint32_t lo = live ? row_starts[s] : 0u, hi = live ? row_starts[s + 1u] : 0u;
        const uint64_t wrong = __ballot(lo > hi || hi > rows);
        const uint64_t from = __ballot(live && lo <= row);
        if (row == 0u && wrong && lane == 0) report(error, kErrAttnRows);
        if (!done && (from | wrong)) {
            done = true;
            const int at = __builtin_ctzll(from | wrong);
            *broken = wrong >> at & 1u;
            if (!*broken && (uint32_t)__builtin_amdgcn_readlane((int)hi, at) > row)
                found = num_seqs - 1u - (base + (uint32_t)at);
        }
        if (done && row != 0u) break;
    }
    return found;
}

// Four e4m3 codes (one dword) as four fp16, exact.
__device__ __forceinline__ uint2 e4m3x4_to_f16(uint32_t w) {
    const h2_t lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
    const h2_t hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
    return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

// Eight query elements, their signs turned by q_sign.
__device__ __forceinline__ uint4 load_query(const uint16_t* p, uint32_t q_sign) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    return make_uint4(u.x ^ q_sign, u.y ^ q_sign, u.z ^ q_sign, u.w ^ q_sign);
}

// --------------------------------------------------- the attention kernels
//
// Both kernels work on the transposed products: S^T = K Q^T (a wave's lanes
// are query rows, its accumulator registers are keys), so a row's running
// maximum and sum stay in its lanes, and P^T leaves the accumulators as the
// second operand of O^T = V^T P^T without a move between lanes: the order in
// which that product takes the keys is free, and V is read in the order in
// which the accumulators hold them. V^T comes out of LDS by transposing reads.
//
// Weights are kept as exp2((x - m) scale_log2 + kWeightBias), x the product q.k
// and m a reference at most kMaxLag powers of two below the row's running
// maximum: a weight's rounding to fp16 is then relative (half a step, 2^-11)
// down to 2^-25 of the largest, and at most 2^15. m moves, and with it the sums,
// only when a logit passes it by kMaxLag. It is a product, not a logit: a
// rounded logit would be off by whole powers of two from 2^24 on, and the
// weight of the very key that it came from with it.
constexpr float kWeightBias = 11.0f;
constexpr float kMaxLag = 4.0f;
// m of a row that has seen no key: below all products (512 x 65504^2), and
// finite times any scale_log2
constexpr float kNoKey = -1e25f;

// Two weights of these exponents, rounded to fp16 for the matrix product. A row's
// sum takes the rounded weights (in fp32): the result is then a mean of the
// values, with the weights off by their rounding, and exact where they are equal.
__device__ __forceinline__ h2_t weight_pair(float x, float y) {
    return h2_t{(_Float16)__builtin_amdgcn_exp2f(x), (_Float16)__builtin_amdgcn_exp2f(y)};
}

// The key tiles (T keys each) that rows at positions p_lo .. p_hi see: those of
// the sinks, then those from the first row's window on. Tile i of them starts
// at key T * key_tile(i).
struct TileSpan {
    uint32_t sink_tiles, first, count;
    __device__ __forceinline__ uint32_t key_tile(uint32_t i) const {
        return i < sink_tiles ? i : first + (i - sink_tiles);
    }
};
template <uint32_t T>
__device__ __forceinline__ TileSpan tile_span(int32_t p_lo, int32_t p_hi, uint32_t window,
                                              uint32_t sinks) {
    TileSpan t{0u, 0u, 0u};
    if (p_hi < 0) return t;
    const uint32_t end = (uint32_t)p_hi / T + 1u;
    if (window && p_lo >= (int32_t)window) {
        t.first = (uint32_t)(p_lo - (int32_t)window + 1) / T;
        const uint32_t s = (sinks + T - 1u) / T;
        t.sink_tiles = s < t.first ? s : t.first;
    }
    t.count = t.sink_tiles + end - t.first;
    return t;
}

// Whether every row at p_lo .. p_hi sees every key of [t, t + T).
template <uint32_t T>
__device__ __forceinline__ bool tile_seen_whole(uint32_t t, int32_t p_lo, int32_t p_hi,
                                                uint32_t window, uint32_t sinks) {
    return (int32_t)(t + T - 1u) <= p_lo &&
           (window == 0u || p_hi - (int32_t)t < (int32_t)window || t + T <= sinks);
}
// Whether any row at p_lo .. p_hi sees any key of [t, t + T).
template <uint32_t T>
__device__ __forceinline__ bool keys_seen(uint32_t t, int32_t p_lo, int32_t p_hi, uint32_t window,
                                          uint32_t sinks) {
    return (int32_t)t <= p_hi &&
           (window == 0u || p_lo - (int32_t)(t + T - 1u) < (int32_t)window || t < sinks);
}
__device__ __forceinline__ bool key_seen(int32_t key, int32_t pos, uint32_t window,
                                         uint32_t sinks) {
    return key <= pos && (window == 0u || pos - key < (int32_t)window || key < (int32_t)sinks);
}

// What a row's sums are multiplied by. A row at a position before 0 is no token,
// sees no key and becomes zeros; any other sees its own key at least, and a sum
// of 0 (all logits -inf) makes it NaN, as 0 / 0.
__device__ __forceinline__ float row_inverse(float sum, int32_t pos, float v_scale) {
    return sum == 0.0f && pos < 0 ? 0.0f : v_scale / sum;
}

// The larger of a lane's value and those of the lanes 32 (and 16) from it.
__device__ __forceinline__ float max_across32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_across16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_across32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float sum_across16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 16 bytes a lane from memory straight into LDS at `lds` + 16 x lane. Issued as
// asm: the compiler would wait for it before any LDS read. It returns no
// register; a wait on vector memory and a barrier come before the data is
// read. m0 is reserved to single instructions (the compiler holds no value in it
// and takes it in no clobber list), and no other here reads it: LDS accesses
// do not from gfx9 on.
__device__ __forceinline__ void dma16(const uint8_t* base, uint32_t lane_off, uint32_t lds) {
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %2"
        :
        : "s"(lds), "v"(lane_off), "s"(base)
        : "memory");
}

// Until at most N of the wave's loads are outstanding (they complete in order),
// and all of its LDS accesses done.
template <uint32_t N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N < 64u, "vmcnt is 6 bits");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// Transposing LDS read: within 16 lanes, lane i gives the address of four
// elements of key i / 4 (elements 4 (i % 4) ..) and gets element i of the four
// keys.
__device__ __forceinline__ uint2 lds_read_tr(const uint8_t* p) {
    typedef short s4_t __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4_t lds_s4_t;
    return __builtin_bit_cast(
        uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)(uintptr_t)p));
}

// Not zero if any element of a dword of the cache is an infinity or NaN: the
// exponent (e4m3: all bits, it has NaN only) of all ones carries into the sign.
template <bool E4M3>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    return E4M3 ? ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u
                : ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
}

typedef _Float16 h4_t __attribute__((ext_vector_type(4)));

// Runs with the plan's device current; the caller's is restored on return.
struct DeviceScope {
    int before = -1;
    hipError_t status = hipSuccess;
    explicit DeviceScope(int device) {
        int now = 0;
        status = hipGetDevice(&now);
        if (status == hipSuccess && now != device) {
            status = hipSetDevice(device);
            if (status == hipSuccess) before = now;
        }
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

constexpr uint64_t kMaxBlocks = (1u << 24) - 1u;  // 256 threads each, under 2^32 in all

// The argument checks every entry point makes, without a device (attn.hip).
tsg_status check_attn_config(const tsg_attn_config* c);
tsg_status check_attn_pages(const tsg_attn_config& c, const tsg_kv_pages* p);
tsg_status check_attn_batch(const tsg_attn_config& c, const tsg_attn_batch* b);
// Whether an attention call may start; fills its kernel's arguments.
tsg_status attn_args(const tsg_attn* attn, const tsg_kv_pages* pages, const tsg_attn_batch* batch,
                     const uint16_t* q, uint32_t q_stride, uint16_t* out, uint32_t out_stride,
                     AttnArgs* a);

// attn_decode.hip
constexpr uint32_t kDecodeTileRows = 16;
constexpr uint32_t kMaxPartials = 2048;  // partial sums (of a 16-row tile) of one call
constexpr uint32_t kMaxPrefillPartials = 512;  // (row tile, key head, split) of one call
constexpr uint32_t kPrefillRows = 128;
// rows of partial results the plan's scratch holds, padded_dim + 2 floats each
constexpr uint32_t kPartialRows = std::max(kMaxPartials * kDecodeTileRows,
                                           kMaxPrefillPartials * kPrefillRows);
tsg_status prepare_decode(const tsg_attn* attn);  // once a plan, its device current
tsg_status launch_decode(const tsg_attn* attn, const AttnArgs& a, tsg_stream stream);
// attn_prefill.hip
tsg_status prepare_prefill(const tsg_attn* attn);
tsg_status launch_prefill(const tsg_attn* attn, const AttnArgs& a, tsg_stream stream);

}  // namespace tsg
